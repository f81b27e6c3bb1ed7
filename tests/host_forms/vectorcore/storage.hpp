// A stand-in for the host's header (see device.hpp).
#pragma once

#include "vectorcore/device.hpp"

#include <cstddef>

namespace vectorcore {

class Storage {
public:
    virtual ~Storage() = default;
    virtual Device device() const noexcept = 0;
    virtual std::size_t size() const noexcept = 0;
};

}  // namespace vectorcore
