// Sizes of the 4-bit cache, in plain C++: what the host lays grids out by.
#pragma once

namespace mxa {

constexpr int kKvBlock = 32;    // tokens of a block
constexpr int kKvMaxDim = 256;  // values of a head

constexpr int kv_groups(int dim) { return (dim + 31) / 32; }

}  // namespace mxa
