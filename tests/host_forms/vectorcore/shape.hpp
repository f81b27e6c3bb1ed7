// A stand-in for the host's header (see device.hpp).
#pragma once

#include <cstddef>
#include <vector>

namespace vectorcore {

using Shape = std::vector<std::size_t>;
using Strides = std::vector<std::size_t>;

inline std::size_t numel(const Shape& shape) {
    std::size_t n = 1;
    for (std::size_t d : shape) n *= d;
    return n;
}

}  // namespace vectorcore
