// A stand-in for the host's header: as much of its interface as
// cuda_backend.hpp is compiled against, for tests that run without the host.
#pragma once

#define VECTORCORE_HAS_CUDA_DEVICE

namespace vectorcore {

struct Device {
    int kind{0};
    static Device cuda() { return Device{2}; }
};

}  // namespace vectorcore
