// What few_kernel of attention.hip reads of keys and values: where a lane's 16 bytes lie, and where the array ends.  Plain arithmetic, for host and device.
#pragma once

#include <cstdint>

namespace tf {
namespace attention {

constexpr uint32_t kOutside = 0x80000000u;  // an offset behind every buffer: reads as zero

// Bytes of a buffer that begins `from` floats into an array of `all`: to the array's end, or as many as an offset may count.  The 16 bytes of a
// row's last columns may reach behind the row; what they reach behind the array is then outside of the buffer, and reads as zero.
constexpr int buffer_bytes(int64_t all, int64_t from) { return all - from < (INT32_MAX / 4) ? (int)((all - from) * 4) : INT32_MAX; }

// Offset of four columns from `column` on of a row, `step` floats behind one another; columns that are none are outside.
constexpr uint32_t buffer_offset(int row, int64_t step, int column, int dim) {
  return column < dim ? (uint32_t)row * (uint32_t)(step * 4) + (uint32_t)column * 4u : kOutside;
}

}  // namespace attention
}  // namespace tf
