// Microscaled 4-bit rows: their layout.
//
// A block is 32 neighbouring values of a row that share a power of two: E2M1 elements
// (0 0.5 1 1.5 2 3 4 6 and their negatives) and one E8M0 byte, 2^(byte - 127). A row of
// `cols` values is P = ceil(cols / 128) groups: 64 * P bytes of codes, two to a byte, the
// even column in the low half; 4 * P scale bytes; zeros up to a multiple of 16. Codes and
// scales past `cols` are zero, so that a product may run over whole groups. A block is 16
// bytes of codes, what one lane feeds the matrix cores' scaled instructions, and a group
// one 32-bit word of scales.
#ifndef GLOW_MI355X_MX4_LAYOUT_H
#define GLOW_MI355X_MX4_LAYOUT_H

#include <cstddef>

namespace mi355x {

constexpr int kMxGroup = 128;       // columns that share a word of scales
constexpr int kMxGroupBytes = 64;   // their codes

inline size_t mx4_groups(size_t cols) { return cols / kMxGroup + (cols % kMxGroup != 0); }
inline size_t mx4_row_bytes_of(size_t cols) { return (mx4_groups(cols) * (kMxGroupBytes + 4) + 15) / 16 * 16; }

} // namespace mi355x

#endif
