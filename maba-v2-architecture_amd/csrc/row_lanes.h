// Where a lane's row is behind its wave's first one, in 32 bits of bytes, for rows that share a wave.  Plain C++, so that the
// arithmetic is tested on the host too.
#pragma once
#include <cstdint>

namespace maba {
namespace rowvec {

// The stride that a tensor of `rows` rows is walked by.  A single row has none: whatever stands for it would put the rows of
// lanes that have no row anywhere.
constexpr int64_t walked(int64_t rows, int64_t stride) { return rows > 1 ? stride : 0; }
// Whether four rows (of at most 4-byte elements) are further apart than 31 bits of bytes tell: such rows have a wave each.
constexpr bool far_apart(int64_t rows, int64_t stride) { return walked(rows, stride) > (int64_t)1 << 27; }
constexpr uint32_t lane_row(int sub, int64_t stride_bytes) { return (uint32_t)(sub * stride_bytes); }

// An offset past every descriptor's end, for lanes without a chunk or a row: it stays there with a lane's own offset added.
constexpr uint32_t NOWHERE = 0x80000000u, DESCRIPTOR_END = 0x7fffffffu;
constexpr uint32_t lane_access(uint32_t lane, uint32_t chunk) { return lane + chunk; }

}  // namespace rowvec
}  // namespace maba
