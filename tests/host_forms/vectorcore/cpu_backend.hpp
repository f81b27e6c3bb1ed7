// A stand-in for the host's header (see device.hpp).
#pragma once

namespace vectorcore::cpu {

enum class BinaryOp { first };
enum class UnaryOp { first };
enum class ReduceOp { first };

}  // namespace vectorcore::cpu
