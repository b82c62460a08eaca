// The paged key / value cache in 4 bits: its layout, shared by the kernels that write, read, move and attend to it.
//
// cache: uint8 [pages, heads, 72 * D]. A block holds 64 tokens of one head: the codes of K (64 rows of D / 2 bytes), the
// parameters of K (64 rows of D / 64 pairs of bf16: scale, zero), then the same of V. A group of 64 channels of a token has a
// scale s, a zero z and codes c in 0..15 and stands for s * c + z:
//   s = bf16((max - min) / 15), z = bf16(min), c = min(15, max(0, rint((x - z) * (1 / s))))
// A row's 32-bit word G w + g (G = D / 64 groups) holds the channels 64 g + 8 w + n in its bits 4 n .. 4 n + 3. So the 8 bytes (4 at
// D = 64) of a lane in a matrix instruction hold eight channels of every group, and no instruction mixes groups.
#pragma once
#include <cstdint>
#include "catcoc/params.h"
#include "catcoc/ptx.cuh"

namespace catcoc {
namespace kv4 {

constexpr int kPage = 64;       // tokens per block
constexpr int kGroup = 64;      // channels per scale and zero
constexpr uint32_t kErrPage = 401u, kErrLen = 402u;   // status word `what`: a page that is not in the cache, a length past the table's row

template <int D>
struct Block {
  static constexpr int kGroups = D / kGroup;
  static constexpr int kRow = D / 2;                        // bytes of a token's codes
  static constexpr int kParRow = 4 * kGroups;               // ... of its scales and zeros
  static constexpr int kPar = kPage * kRow;                 // offset of the parameters behind the codes
  static constexpr int kHalf = kPage * (kRow + kParRow);    // K's half of the block, then V's
  static constexpr int kBytes = 2 * kHalf;
};

// A bad argument that only the device can see: recorded once, the access is left out.
CATCOC_DEVICE void note(uint32_t* status, uint32_t what, int seen, int limit) {
  if (atomicCAS(status, 0u, static_cast<uint32_t>(STATUS_BAD_ARGUMENT)) == 0u) {
    status[1] = 0u; status[2] = what; status[3] = static_cast<uint32_t>(limit); status[4] = static_cast<uint32_t>(seen); status[5] = 0u;
    status[6] = blockIdx.x;
    __threadfence_system();
  }
}

// Length of a sequence, cut to what its row of the block table can hold
CATCOC_DEVICE int seq_len(const int* lens, int b, int capacity, uint32_t* status) {
  const int n = lens[b];
  if (n < 0 || n > capacity) {
    note(status, kErrLen, n, capacity);
    return n < 0 ? 0 : capacity;
  }
  return n;
}

// A block table's entry, -1 where it names no page
CATCOC_DEVICE int checked_page(int page, int pages, uint32_t* status) {
  if (static_cast<uint32_t>(page) < static_cast<uint32_t>(pages)) return page;
  note(status, kErrPage, page, pages);
  return -1;
}
// Page `i` of a sequence, or -1
CATCOC_DEVICE int page_of(const int* table, int64_t row, int i, int pages, uint32_t* status) { return checked_page(table[row + i], pages, status); }

CATCOC_DEVICE float bf16_lo(uint32_t pair) { return __uint_as_float(pair << 16); }
CATCOC_DEVICE float bf16_hi(uint32_t pair) { return __uint_as_float(pair & 0xffff0000u); }

}  // namespace kv4
}  // namespace catcoc
