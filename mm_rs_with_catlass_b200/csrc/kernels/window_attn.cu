// Causal flash attention with a sliding window and visible first keys (sinks) on tcgen05: flash_attn.cu's tile, walked by a persistent CTA.
//
// A tile of 128 query rows sees window + 128 keys at most, a few blocks of 128, where a causal tile sees up to all of them. So
// what a CTA does besides its blocks counts: with a launch's CTAs one after the other, 1 x 32 / 8 heads x 8192 took 1.67 us a block and
// 8.3 us a CTA (TMEM, barriers, the first copies and products, the last ones, the store). Here an SM keeps one CTA, which
// takes every 148th piece of work: the copies run on into the next one, its first scores are computed under the last block's end, and the
// output leaves by TMA while it is worked on. (First scores ahead of the last block's product with V waited for the next queries: 117 -> 124 us.)
//
//   warps 0..3, 4..7  softmax of tile 0, tile 1: one query row per thread (softmax_row.cuh)
//   warp 8            TMA producer: Q tiles, K and V blocks of 128 keys through one ring of slots
//   warp 9 (, 10)     MMA issuer; at D = 128 one for each tile
//
// A piece of work is two tiles of a head and the list of the blocks that their rows see: those of the sinks, then from the first block
// that some row's window reaches. Both tiles walk the list from its start; a block in front of tile 1's windows stands behind the blocks of
// both and ahead of tile 1's last one, and tile 1 leaves it out, so that both walk as many blocks as they see, in step.
//
// TMEM columns, D = 128: one buffer of scores for both tiles [0, 128), P_0 and P_1 at 128 and 192, O_0 and O_1 at 256 and 384. D = 64:
// S_0, S_1 at 0 and 128, O_0, O_1 at 256 and 320, P_0, P_1 at 384 and 448.
//
// The recurrence and its rounding are flash_attn.cu's: P = exp2(scale S - m) in the operands' type, m moved only when some row exceeds it by 8.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <algorithm>
#include <cstring>
#include <type_traits>
#include "catcoc/attn_host.h"
#include "catcoc/capi.h"
#include "catcoc/host_util.h"
#include "catcoc/params.h"
#include "catcoc/ptx.cuh"
#include "catcoc/slices.cuh"
#include "catcoc/softmax_row.cuh"

namespace catcoc {
namespace window {

using attn::RowState;
using attn::pack16;

constexpr int kBQ = 128, kTiles = 2, kBKV = 128;
constexpr int kThreads = 384;
constexpr int kSoftmaxRegs = 216, kOtherRegs = 72;   // of 168 a thread: 2 x 216 + 72 = 3 x 168
constexpr int kProducerWarp = 8, kIssuerWarp = 9;
constexpr int kBlockBytes = 128 * 128;               // one 128-row x 128-byte (64 element) swizzled block
constexpr int kMaxSlots = 8;
constexpr int kOutBytes = 8 * 32 * 128;

// Division of numbers below 2^31 by a number that the host knows: n / d = n m >> (31 + s) with d <= 2^s and m = 2^(31 + s) / d + 1. The
// divisions of a piece of work were a chain of thousands of cycles in front of its first block (window 128: 11.1 us a piece).
struct Divisor {
  uint32_t d, m, s;
  void set(uint32_t by) {
    d = by;
    for (s = 0; (1u << s) < by; ++s) {}
    m = static_cast<uint32_t>((1ull << (31 + s)) / by + 1ull);
  }
  CATCOC_DEVICE int div(int n) const { return static_cast<int>((static_cast<uint64_t>(static_cast<uint32_t>(n)) * m) >> (31u + s)); }
  CATCOC_DEVICE int mod(int n) const { return n - div(n) * static_cast<int>(d); }
};

struct WindowParams {
  CUtensorMap tm_q, tm_k, tm_v;   // {D, S, B * H} with a {64, 128, 1} box, 128-byte swizzle
  CUtensorMap tm_o;               // out {D, Sq, B * Hq} with a {64, 32, 1} box: a warp's rows, of which those past Sq are not written
  int B, Hq, Hk, Sq, Sk;          // Sq: rows per (batch, query head), or per (batch, KV head) when its heads are packed
  int pos;                        // query positions: row r stands at r % pos
  int window, sinks;
  int tiles, works, slices;       // pieces of work a head, in all, and slices of each
  Divisor by_works, by_heads, by_hq, by_group, by_pos;   // works, B * Hq, Hq, Hq / Hk, pos
  float scale_log2;               // softmax scale * log2(e), > 0
  uint32_t idesc_qk, idesc_pv;
  uint32_t* status;
  uint64_t timeout_ns;
  float* part_o;                  // keys cut into slices: [slice][B * Hq * Sq][D] unnormalised pieces
  float* part_ml;                 // [slice][B * Hq * Sq][2]
  int per;                        // items of a slice
};

struct Bars {
  uint64_t q_full[kTiles], q_empty[kTiles], kv_full[kMaxSlots], kv_empty[kMaxSlots], s_full[kTiles], s_free[kTiles], p_half[kTiles], p_full[kTiles], pv_done[kTiles];
  uint64_t drain[2];                               // of an issuer whose launch was given up: its products have retired
  uint32_t tmem_base, abort_flag, kv_sent, q_sent[kTiles];
};

CATCOC_DEVICE void fail(const WindowParams& p, uint32_t what, uint32_t a) {
  if (atomicCAS(p.status, 0u, static_cast<uint32_t>(STATUS_TIMEOUT_PIPELINE)) == 0u) {
    p.status[1] = 0u; p.status[2] = 500u + what; p.status[3] = a; p.status[4] = 0u; p.status[5] = 0u;
    p.status[6] = blockIdx.x;
    __threadfence_system();
  }
}

// A piece of work and its list of blocks ("items")
template <bool CUT>
struct Work {
  int bh, bhk, q0, slice;
  int nblk[kTiles], items;                 // blocks a tile walks, and of the list
  int first, sink_blocks, shared, j0;
  bool skip;                               // tile 1 leaves out the item `shared`, the last one of tile 0
  int lo[kTiles], hi[kTiles];              // positions of a tile's rows

  CATCOC_DEVICE Work(const WindowParams& p, int index) {
    slice = CUT ? p.by_works.div(index) : 0;
    const int w = index - slice * p.works, heads = p.B * p.Hq;
    // heads side by side, so that those of a KV head meet its blocks in the L2; the early tiles, which see less, last
    const int early = p.by_heads.div(w), qt = p.tiles - 1 - early;
    bh = w - early * heads;
    q0 = qt * (kTiles * kBQ);
    const int b = p.by_hq.div(bh);
    bhk = b * p.Hk + p.by_group.div(bh - b * p.Hq);
    const int shift = p.Sk - p.pos;
#pragma unroll
    for (int t = 0; t < kTiles; ++t) {
      // (all positions when the rows of two packed heads meet in the tile; a tile without rows does as the other)
      const int r = p.by_pos.mod(q0 + (t == 1 && q0 + kBQ >= p.Sq ? 0 : t * kBQ));
      const bool wrap = r + kBQ > p.pos && p.pos < p.Sq;
      lo[t] = (wrap ? 0 : r) + shift;
      hi[t] = min(wrap ? p.pos - 1 : r + kBQ - 1, p.pos - 1) + shift;
      nblk[t] = hi[t] / kBKV + 1;
    }
    const int first0 = max(0, lo[0] - p.window + 1) / kBKV, first1 = max(0, lo[1] - p.window + 1) / kBKV, want = (p.sinks + kBKV - 1) / kBKV;
    first = min(first0, first1);
    sink_blocks = min(want, first);
    skip = !CUT && first1 == first + 1 && nblk[1] == nblk[0] + 1 && first >= want;
    shared = sink_blocks + nblk[0] - first - 1;
    j0 = CUT ? slice * p.per : 0;
#pragma unroll
    for (int t = 0; t < kTiles; ++t) {
      nblk[t] += sink_blocks - first - (skip && t == 1 ? 1 : 0);
      // (a slice that some tile sees nothing of is a masked block there: a maximum of -inf, a sum of zero)
      if constexpr (CUT) nblk[t] = max(1, min(p.per, nblk[t] - j0));
    }
    nblk[1] = max(nblk[0], nblk[1]);
    items = nblk[1] + (skip ? 1 : 0);
  }
  CATCOC_DEVICE int block_of(int item) const {
    item += j0;
    if (item < sink_blocks) return item;
    if (!skip) return first + item - sink_blocks;
    return item == shared ? first : first + item - sink_blocks + (item < shared ? 1 : 0);
  }
  // The tile's blocks that all of its rows see whole: the first `sinks_end` and [begin, end) of those it walks, at least
  CATCOC_DEVICE void whole(const WindowParams& p, int t, int& sinks_end, int& begin, int& end) const {
    const int ahead = sink_blocks - first - (skip ? 1 : 0) - j0;         // walked as the (block + ahead)-th
    sinks_end = min(p.sinks / kBKV, sink_blocks) - j0;
    begin = max(sink_blocks - j0, (hi[t] >= p.window ? (hi[t] - p.window) / kBKV + 1 : 0) + ahead);
    end = (lo[t] + 1) / kBKV + ahead;
  }
  CATCOC_DEVICE int item_of(int t, int j) const { return skip && t == 1 && j == shared ? j + 1 : j; }
};

template <int D, int FMT, bool CUT>
__global__ void __launch_bounds__(kThreads, 1) window_attn_kernel(const __grid_constant__ WindowParams p) {
  constexpr int kDB = D / 64;                    // 128-byte blocks along the head dimension
  constexpr int kQBytes = kDB * kBlockBytes;     // one Q tile
  constexpr int kSlotBytes = kDB * kBlockBytes;  // one K or V block: 128 keys x D
  constexpr int kSlots = D == 128 ? 4 : 8;       // ring of K / V blocks (K_0 V_0 K_1 V_1 ...), running on over the pieces of work
  constexpr uint32_t kTmemCols = 512;
  constexpr uint32_t kOCol = 256;
  constexpr bool kOneS = D == 128;
  constexpr int kIssuers = kOneS ? 2 : 1;
  constexpr uint32_t kPCol = kOneS ? 128 : 384;    // P_t at kPCol + t * 64
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~static_cast<uintptr_t>(1023));
  uint8_t* sq = smem;                            // two Q tiles
  uint8_t* skv = sq + kTiles * kQBytes;
  uint8_t* sout = skv + kSlots * kSlotBytes;     // of each softmax warp, 32 rows x 64 columns on their way out
  Bars* bars = reinterpret_cast<Bars*>(sout + kOutBytes);
  volatile uint32_t* abort_flag = &bars->abort_flag;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int total = p.works * p.slices;

  if (threadIdx.x == 0) {
    for (int s = 0; s < kSlots; ++s) { ptx::mbar_init(&bars->kv_full[s], 1); ptx::mbar_init(&bars->kv_empty[s], kIssuers); }
    for (int t = 0; t < kTiles; ++t) {
      ptx::mbar_init(&bars->drain[t], 1);
      bars->q_sent[t] = 0;
      ptx::mbar_init(&bars->q_full[t], 1);
      ptx::mbar_init(&bars->q_empty[t], 1);
      ptx::mbar_init(&bars->s_full[t], 1);
      ptx::mbar_init(&bars->s_free[t], 4);
      ptx::mbar_init(&bars->pv_done[t], 1);
      ptx::mbar_init(&bars->p_half[t], 4);         // one arrival per softmax warp: P of the first 64 keys is in TMEM
      ptx::mbar_init(&bars->p_full[t], 4);         // ... of all of them
    }
    bars->abort_flag = 0;
    bars->kv_sent = 0;
    ptx::mbar_fence_init();
    ptx::prefetch_tmap(&p.tm_q); ptx::prefetch_tmap(&p.tm_k); ptx::prefetch_tmap(&p.tm_v);
  }
  if (warp == kIssuerWarp) { ptx::tmem_alloc(&bars->tmem_base, kTmemCols); ptx::tmem_relinquish(); }
  ptx::tcgen05_fence_before();
  __syncthreads();
  ptx::tcgen05_fence_after();
  const uint32_t tmem = bars->tmem_base;
  ptx::grid_dependency_wait();
  if constexpr (CUT) ptx::launch_dependents();                       // the merge waits for this grid's results by itself

  if (warp >= kProducerWarp) ptx::reg_dec<kOtherRegs>();   // all four warps of the warpgroup at one place
  if (warp == kProducerWarp) {
    // ------------------------------ TMA producer ------------------------------
    // item 2 x is the K block and 2 x + 1 the V block of the x-th block since the start; item i lives in slot i % kSlots
    bool ok = true;
    uint32_t count = 0, base = 0;                  // pieces of work, items before this one
    for (int index = blockIdx.x; ok && index < total; index += gridDim.x, ++count) {
      const Work<CUT> w(p, index);
      for (int t = 0; ok && t < kTiles; ++t) {
        ok = ptx::mbar_wait(&bars->q_empty[t], (count & 1u) ^ 1u, p.timeout_ns, abort_flag);
        if (ok && ptx::elect_one()) {
          bars->q_sent[t] = count + 1u;
          ptx::mbar_expect_tx(&bars->q_full[t], kQBytes);
          for (int d = 0; d < kDB; ++d) ptx::tma_load_3d(sq + t * kQBytes + d * kBlockBytes, &p.tm_q, &bars->q_full[t], d * 64, w.q0 + t * kBQ, w.bh);
        }
        __syncwarp();
      }
      for (int i = 0; ok && i < 2 * w.items; ++i) {
        const uint32_t item = base + static_cast<uint32_t>(i), slot = item % kSlots;
        ok = ptx::mbar_wait(&bars->kv_empty[slot], ((item / kSlots) & 1u) ^ 1u, p.timeout_ns, abort_flag);
        if (ok && ptx::elect_one()) {
          bars->kv_sent = item + 1u;
          ptx::mbar_expect_tx(&bars->kv_full[slot], kSlotBytes);
          const CUtensorMap* tm = (i & 1) ? &p.tm_v : &p.tm_k;
          for (int d = 0; d < kDB; ++d)
            ptx::tma_load_3d(skv + slot * kSlotBytes + d * kBlockBytes, tm, &bars->kv_full[slot], d * 64, w.block_of(i >> 1) * kBKV, w.bhk);
        }
        __syncwarp();
      }
      base += 2u * static_cast<uint32_t>(w.items);
    }
    if (!ok && lane == 0) { fail(p, 1u, 0u); *abort_flag = 1; }
  } else if (warp >= kIssuerWarp && warp < kIssuerWarp + kIssuers) {
    // ------------------------------ MMA issuers ------------------------------
    const uint64_t dq0 = ptx::make_smem_desc_sw128(ptx::smem_u32(sq), 16u, 1024u);
    const uint64_t dk0 = ptx::make_smem_desc_sw128(ptx::smem_u32(skv), 16u, 1024u);
    const uint64_t dv0 = ptx::make_smem_desc_sw128(ptx::smem_u32(skv), static_cast<uint32_t>(kBlockBytes), 1024u);
    // (addresses are in the low words, which no tile or slot carries over into the high ones)
    const uint32_t q_lo = static_cast<uint32_t>(dq0), q_hi = static_cast<uint32_t>(dq0 >> 32);
    const uint32_t k_lo = static_cast<uint32_t>(dk0), k_hi = static_cast<uint32_t>(dk0 >> 32);
    const uint32_t v_lo = static_cast<uint32_t>(dv0), v_hi = static_cast<uint32_t>(dv0 >> 32);
    // what came before a piece of work: pieces, items, and blocks that either tile walked
    struct Before { uint32_t count, base, c[kTiles]; };
    auto wait_item = [&](uint32_t item) { return ptx::mbar_wait(&bars->kv_full[item % kSlots], (item / kSlots) & 1u, p.timeout_ns, abort_flag); };
    // An item that a tile leaves out is handed back for it once it has arrived (D = 128, where both tiles' issuers hand back each one)
    auto pass = [&](uint32_t item) {
      if (!wait_item(item)) return false;
      if (lane == 0) ptx::mbar_arrive(&bars->kv_empty[item % kSlots]);
      return true;
    };
    // Who hands an item back at D = 64: the tile that uses it last
    auto last_use = [&](const Work<CUT>& w, int t, int j) { return kOneS || t == 1 || (w.skip && j == w.shared); };
    // S_t[128, 128 keys] = Q_t[128, D] K^T of the tile's j-th block, behind the softmax's read of what is in the buffer: both
    // operands K-major (D contiguous), 16 elements of D per MMA
    auto scores = [&](const Work<CUT>& w, const Before& f, int t, int j) {
      const int x = w.item_of(t, j);
      if (kOneS && x != j && !pass(f.base + 2u * static_cast<uint32_t>(j))) return false;
      const uint32_t item = f.base + 2u * static_cast<uint32_t>(x);
      if (j == 0 && !ptx::mbar_wait(&bars->q_full[t], f.count & 1u, p.timeout_ns, abort_flag)) return false;
      if (!wait_item(item)) return false;
      // The block that was in the buffer before: at D = 128 the tiles take it in turn, and tile 1 by itself behind tile 0's last one
      const int tile = !kOneS ? t : (t == 1 && j < w.nblk[0] ? 0 : 1);
      const uint32_t before = f.c[tile] + static_cast<uint32_t>(j) + (tile == 0 && t == 1 ? 1u : 0u);   // blocks of that tile until then
      if (before > 0u && !ptx::mbar_wait(&bars->s_free[tile], (before - 1u) & 1u, p.timeout_ns, abort_flag)) return false;
      ptx::tcgen05_fence_after();
      const uint32_t slot = item % kSlots;
      if (ptx::elect_one()) {
        const uint32_t ql = q_lo + static_cast<uint32_t>(t * (kQBytes >> 4)), kl = k_lo + slot * (kSlotBytes >> 4);
#pragma unroll
        for (int kk = 0; kk < D / 16; ++kk) {
          const uint32_t off = static_cast<uint32_t>(((kk >> 2) * kBlockBytes + (kk & 3) * 32) >> 4);
          ptx::umma_f16(tmem + (kOneS ? 0 : t * 128), ptx::desc_of(ql + off, q_hi), ptx::desc_of(kl + off, k_hi), p.idesc_qk, kk != 0 ? 1u : 0u);
        }
        ptx::tcgen05_commit(&bars->s_full[t]);
        if (last_use(w, t, j)) ptx::tcgen05_commit(&bars->kv_empty[slot]);
        if (j + 1 == w.nblk[t]) ptx::tcgen05_commit(&bars->q_empty[t]);
      }
      __syncwarp();
      return true;
    };
    // O_t[128, D] += P_t[128, 128 keys] V[128 keys, D]: P from TMEM (row = lane, two keys per 32-bit column, 8 columns per MMA), V
    // MN-major (D contiguous): 16 key rows per MMA = 2048 bytes down a block, blocks of 64 head-dim columns 16 KiB apart
    auto values = [&](const Work<CUT>& w, const Before& f, int t, int j) {
      const int x = w.item_of(t, j);
      if (kOneS && x != j && !pass(f.base + 2u * static_cast<uint32_t>(j) + 1u)) return false;
      const uint32_t item = f.base + 2u * static_cast<uint32_t>(x) + 1u, slot = item % kSlots;
      const uint32_t vl = v_lo + slot * (kSlotBytes >> 4), c = f.c[t] + static_cast<uint32_t>(j);
      if (!wait_item(item)) return false;
      constexpr int kParts = kOneS ? 1 : 2, kPerPart = kBKV / 16 / kParts;
#pragma unroll
      for (int part = 0; part < kParts; ++part) {
        if (!ptx::mbar_wait(part + 1 < kParts ? &bars->p_half[t] : &bars->p_full[t], c & 1u, p.timeout_ns, abort_flag)) return false;
        ptx::tcgen05_fence_after();
        if (ptx::elect_one()) {
#pragma unroll
          for (int kk = part * kPerPart; kk < (part + 1) * kPerPart; ++kk)
            ptx::umma_f16_ts(tmem + kOCol + t * D, tmem + kPCol + t * 64 + kk * 8, ptx::desc_of(vl + static_cast<uint32_t>((kk * 16 * 128) >> 4), v_hi),
                             p.idesc_pv, (j > 0 || kk != 0) ? 1u : 0u);
          if (part + 1 == kParts) {
            ptx::tcgen05_commit(&bars->pv_done[t]);
            if (last_use(w, t, j)) ptx::tcgen05_commit(&bars->kv_empty[slot]);
          }
        }
        __syncwarp();
      }
      return true;
    };
    bool ok = true;
    Before f{0u, 0u, {0u, 0u}};
    for (int index = blockIdx.x; ok && index < total; index += gridDim.x) {
      const Work<CUT> w(p, index);
      if constexpr (kOneS) {
        const int t = warp - kIssuerWarp, nt = w.nblk[t];
        ok = scores(w, f, t, 0);
        for (int j = 0; ok && j < nt; ++j) {
          if (j + 1 < nt) ok = scores(w, f, t, j + 1);      // ahead of the product with V, which waits for this block's softmax
          ok = ok && values(w, f, t, j);
        }
        // items behind tile 0's last one
        for (int i = 2 * nt; ok && t == 0 && i < 2 * w.items; ++i) ok = pass(f.base + static_cast<uint32_t>(i));
      } else {
        ok = scores(w, f, 0, 0) && scores(w, f, 1, 0);
        for (int j = 0; ok && j < w.nblk[1]; ++j) {
#pragma unroll
          for (int t = 0; t < kTiles; ++t)
            if (j + 1 < w.nblk[t]) ok = ok && scores(w, f, t, j + 1);
#pragma unroll
          for (int t = 0; t < kTiles; ++t)
            if (j < w.nblk[t]) ok = ok && values(w, f, t, j);
        }
      }
      ++f.count;
      f.base += 2u * static_cast<uint32_t>(w.items);
      f.c[0] += static_cast<uint32_t>(w.nblk[0]);
      f.c[1] += static_cast<uint32_t>(w.nblk[1]);
    }
    if (!ok && lane == 0) { fail(p, 2u, 0u); *abort_flag = 1; }
  } else if (warp < kProducerWarp) {
    // ------------------------------ softmax / correction / epilogue ------------------------------
    ptx::reg_inc<kSoftmaxRegs>();
    const int t = warp >> 2;                         // query tile of this warp
    const int qd = warp & 3;                         // TMEM lane quarter of this warp
    const uint32_t t_lane = tmem + (static_cast<uint32_t>(qd * 32) << 16);
    const uint32_t t_s = t_lane + (kOneS ? 0 : t * 128), t_p = t_lane + kPCol + t * 64, t_o = t_lane + kOCol + t * D;
    const float sc = p.scale_log2;
    bool ok = true;
    uint32_t c = 0;                                  // blocks of this tile since the start
    for (int index = blockIdx.x; ok && index < total; index += gridDim.x) {
      // (only what every block needs stays in registers, which hold the row's 128 scores; the rest is worked out where it is needed)
      int n_mine, sinks_end, begin, end;
      {
        const Work<CUT> w(p, index);
        n_mine = w.nblk[t];
        w.whole(p, t, sinks_end, begin, end);
      }
      auto again = [&] {
        int same = index;
        asm volatile("" : "+r"(same));
        return Work<CUT>(p, same);
      };
      RowState st;
      for (int j = 0; j < n_mine; ++j, ++c) {
        if (!ptx::mbar_wait(&bars->s_full[t], c & 1u, p.timeout_ns, abort_flag)) { ok = false; break; }
        ptx::tcgen05_fence_after();
        // P V of the block before has read P, and O is whole
        auto previous = [&] {
          if (j > 0 && !ptx::mbar_wait(&bars->pv_done[t], (c - 1u) & 1u, p.timeout_ns, abort_flag)) ok = false;
          ptx::tcgen05_fence_after();
        };
        const bool masked = j >= sinks_end && (j < begin || j >= end);
        auto mask = [&] {
          const Work<CUT> w = again();
          const int key0 = w.block_of(w.item_of(t, j)) * kBKV, mine = p.by_pos.mod(w.q0 + t * kBQ + qd * 32 + lane) + p.Sk - p.pos;
          return attn::WindowMask(mine + 1 - key0, mine - p.window + 1 - key0, p.sinks - key0);
        };
        attn::softmax_row_block<FMT>(t_s, t_p, masked, mask, sc, st, [&] {
          ptx::tcgen05_fence_before();
          __syncwarp();
          if (lane == 0) ptx::mbar_arrive(&bars->s_free[t]);
        }, [&](bool move, float alpha) {
          if (move) previous();
          if (move && j > 0) attn::rescale_o<D>(t_o, alpha);
        }, [&] { previous(); }, [&] {
          if constexpr (!kOneS) {
            ptx::tcgen05_wait_st();
            ptx::tcgen05_fence_before();
            __syncwarp();
            if (lane == 0) ptx::mbar_arrive(&bars->p_half[t]);
          }
        });
        ok = __all_sync(0xffffffffu, ok);
        if (!ok) break;
        ptx::tcgen05_wait_st();
        ptx::tcgen05_fence_before();
        __syncwarp();
        if (lane == 0) ptx::mbar_arrive(&bars->p_full[t]);
      }
      if (ok) ok = ptx::mbar_wait(&bars->pv_done[t], (c - 1u) & 1u, p.timeout_ns, abort_flag);
      ok = __all_sync(0xffffffffu, ok);
      if (!ok) break;
      ptx::tcgen05_fence_after();
      const float inv = (st.l > 0.0f) ? 1.0f / st.l : 0.0f;
      const Work<CUT> w = again();
      const int row0 = w.q0 + t * kBQ + qd * 32;           // this warp's first query row inside the head
#pragma unroll
      for (int col = 0; col < D / 32; ++col) {
        uint32_t v[32];
        ptx::tmem_ld_32x32b_x32(t_o + col * 32, v);
        ptx::tcgen05_wait_ld();
        if constexpr (CUT) {
          if (row0 + lane < p.Sq) {
            const int64_t prow = (static_cast<int64_t>(w.slice) * p.B * p.Hq + w.bh) * p.Sq + row0 + lane;
#pragma unroll
            for (int u = 0; u < 8; ++u) ptx::st_global_v4(p.part_o + prow * D + col * 32 + u * 4, make_uint4(v[u * 4], v[u * 4 + 1], v[u * 4 + 2], v[u * 4 + 3]));
            if (col == 0) *reinterpret_cast<float2*>(p.part_ml + prow * 2) = make_float2(st.m, st.l);
          }
        } else {
          // 64 columns at a time through shared memory (its 128-byte swizzle is the map's) and out by one copy: stores of a row a thread
          // took 2.5 us of every piece (1 x 32 / 8 x 8192, window 1024: 150 us, without any stores 136)
          const uint32_t at = ptx::smem_u32(sout + warp * 4096) + static_cast<uint32_t>(lane * 128);
          if ((col & 1) == 0) {
            if (lane == 0) ptx::bulk_wait_group_read<0>();  // the copy before has read the place
            __syncwarp();
          }
#pragma unroll
          for (int u = 0; u < 4; ++u) {
            uint32_t x[4];
#pragma unroll
            for (int e = 0; e < 4; ++e)
              x[e] = pack16<FMT>(__uint_as_float(v[u * 8 + 2 * e]) * inv, __uint_as_float(v[u * 8 + 2 * e + 1]) * inv);
            ptx::st_shared_v4(at + static_cast<uint32_t>(((((col & 1) * 4 + u) ^ (lane & 7)) * 16)), make_uint4(x[0], x[1], x[2], x[3]));
          }
          if ((col & 1) == 1) {
            ptx::fence_proxy_async_smem();
            __syncwarp();
            if (lane == 0 && row0 < p.Sq) {
              ptx::tma_store_3d(&p.tm_o, ptx::smem_u32(sout + warp * 4096), (col >> 1) * 64, row0, w.bh);
              ptx::bulk_commit_group();
            }
          }
        }
      }
      // (the next piece's first product with V overwrites O behind this warp's arrival at p_full, which follows these reads)
      ptx::tcgen05_fence_before();
    }
    if (!ok && lane == 0) { fail(p, 3u, t); *abort_flag = 1; }
    if (!CUT && lane == 0) ptx::bulk_wait_group_all();      // what is on its way out has been read and written
  }

  ptx::tcgen05_fence_before();
  __syncthreads();
  if (*abort_flag != 0) {
    // the launch was given up: copies on their way land, and products retire, before the block's memory is handed on
    volatile uint32_t never = 0;
    if (warp == kProducerWarp) {
      const uint32_t sent = bars->kv_sent;
      for (uint32_t i = sent > kSlots ? sent - kSlots : 0u; i < sent; ++i) ptx::mbar_wait(&bars->kv_full[i % kSlots], (i / kSlots) & 1u, 100000000ull, &never);
      for (int t = 0; t < kTiles; ++t)
        if (bars->q_sent[t] != 0u) ptx::mbar_wait(&bars->q_full[t], (bars->q_sent[t] - 1u) & 1u, 100000000ull, &never);
    } else if (warp >= kIssuerWarp && warp < kIssuerWarp + kIssuers) {
      if (ptx::elect_one()) ptx::tcgen05_commit(&bars->drain[warp - kIssuerWarp]);
      __syncwarp();
      ptx::mbar_wait(&bars->drain[warp - kIssuerWarp], 0u, 100000000ull, &never);
    }
    __syncthreads();
  }
  ptx::tcgen05_fence_after();
  if (warp == kIssuerWarp) ptx::tmem_dealloc(tmem, kTmemCols);
}

}  // namespace window
}  // namespace catcoc

using namespace catcoc;
using namespace catcoc::host;

namespace {
struct WindowPlan {
  int Hq, Sq;          // as the kernel sees them (the query heads of a KV head may be packed)
  int tiles;
  int slices, per;     // keys cut into slices of `per` blocks
};

WindowPlan window_plan(int B, int Hq, int Hk, int Sq, int Sk, int window, int sinks, int sms) {
  const int group = Hq / Hk, rows = window::kTiles * window::kBQ, pos = Sq;
  // blocks of the list of `span` positions that end before key `end`, at most (Work: those of the sinks are whole ones)
  auto blocks = [&](int64_t end, int span) {
    const int64_t most = static_cast<int64_t>(window) + span + 126 + (static_cast<int64_t>(sinks) + 127) / 128 * 128;
    return static_cast<int>((std::min<int64_t>(end, most) + 127) / 128);
  };
  struct Form { WindowPlan plan; int longest; double load; } forms[2];
  // In units of a block: a piece of work takes its blocks and about one more for its ends. A launch takes its total over the SMs, or
  // its longest piece.
  auto form = [&](int hq, int sq, int span) {
    Form f{{hq, sq, (sq + rows - 1) / rows, 1, 0}, blocks(Sk, span), 0.0};
    double sum = 0.0;
    for (int i = 0; i < f.plan.tiles; ++i) sum += 1.0 + blocks(span == pos ? Sk : std::min<int64_t>(Sk, static_cast<int64_t>(i + 1) * rows + Sk - pos), span);
    f.load = std::max(1.0 + f.longest, static_cast<double>(B) * hq * sum / sms);
    return f;
  };
  int n = 1;
  forms[0] = form(Hq, Sq, std::min(rows, pos));
  // the query heads of a KV head are contiguous rows: with few positions they fill tiles together (a tile may then span all positions)
  if (group > 1 && static_cast<int64_t>(group) * Sq <= (1 << 24)) forms[n++] = form(Hk, group * Sq, pos);
  WindowPlan best = n > 1 && forms[1].load < 0.95 * forms[0].load ? forms[1].plan : forms[0].plan;
  // Few pieces over long windows leave SMs idle: the lists are cut, and a second kernel merges (the rule and its figures: flash_attn.cu)
  const double longest = std::min(forms[0].longest, n > 1 ? forms[1].longest : forms[0].longest);
  if (longest < 14.0) return best;
  double best_us = 0.85 * (5.0 + 1.55 * longest);
  for (int f = 0; f < n; ++f) {
    const WindowPlan& x = forms[f].plan;
    const int64_t works = static_cast<int64_t>(B) * x.Hq * x.tiles, out_rows = static_cast<int64_t>(B) * x.Hq * x.Sq;
    for (int s = 2; s <= 16 && works * s <= sms && 2 * s <= forms[f].longest; ++s) {
      const int per = (forms[f].longest + s - 1) / s, slices = (forms[f].longest + per - 1) / per;
      const double us = 9.0 + 1.55 * per + static_cast<double>(slices) * out_rows * 128 * 8 / 3e6;
      if (us < best_us) { best_us = us; best = x; best.slices = slices; best.per = per; }
    }
  }
  return best;
}

int current_sms() {
  int device = 0;
  cudaGetDevice(&device);
  return catcoc_num_sms(device);
}

bool window_args(int B, int Hq, int Hk, int Sq, int Sk, int D, int window, int sinks) {
  return B > 0 && Hq > 0 && Hk > 0 && Sq > 0 && Sk >= Sq && Hq % Hk == 0 && (D == 64 || D == 128) && window >= 1 && sinks >= 0;
}
}  // namespace

extern "C" int64_t catcoc_window_route(int B, int Hq, int Hk, int Sq, int Sk, int D, int window, int sinks) {
  if (!window_args(B, Hq, Hk, Sq, Sk, D, window, sinks)) return -1;
  window = std::min(window, 1 << 30);
  sinks = std::min(sinks, 1 << 30);
  const int64_t decode = catcoc_window_decode_workspace_bytes(B, Hq, Hk, Sq, Sk, D, window, sinks);
  if (decode >= 0) return decode;
  const WindowPlan d = window_plan(B, Hq, Hk, Sq, Sk, window, sinks, current_sms());
  return -1 - (d.slices > 1 ? static_cast<int64_t>(d.slices) * B * Hq * Sq * (D + 2) * static_cast<int64_t>(sizeof(float)) : 0);
}

extern "C" int catcoc_window_attention(const void* q, const void* k, const void* v, void* out, void* workspace, int B, int Hq, int Hk, int Sq, int Sk, int D,
                                       int fmt, int window, int sinks, float scale, uint32_t* status, uint64_t timeout_ns, void* stream_) {
  if (!q || !k || !v || !out || !status || !window_args(B, Hq, Hk, Sq, Sk, D, window, sinks)) {
    set_error("window_attention: bad arguments (D 64 or 128, Sk >= Sq, a window of at least 1, no negative sinks)");
    return CATCOC_E_BAD_ARG;
  }
  if (fmt != CATCOC_FMT_F16 && fmt != CATCOC_FMT_BF16) { set_error("flash_attention takes fp16 / bf16"); return CATCOC_E_UNSUPPORTED; }
  if (!(scale > 0.0f)) { set_error("flash_attention: the softmax scale must be positive (the row maximum is taken before scaling)"); return CATCOC_E_UNSUPPORTED; }
  window = std::min(window, 1 << 30);                              // (both beyond any length; their sums stay in range)
  sinks = std::min(sinks, 1 << 30);
  if (catcoc_window_decode_workspace_bytes(B, Hq, Hk, Sq, Sk, D, window, sinks) >= 0)
    return catcoc_window_decode(q, k, v, out, workspace, B, Hq, Hk, Sq, Sk, D, fmt, window, sinks, scale, status, timeout_ns, stream_);
  const int pos = Sq;
  const int sms = current_sms();
  const WindowPlan d = window_plan(B, Hq, Hk, Sq, Sk, window, sinks, sms);
  if (d.slices > 1 && workspace == nullptr) { set_error("window_attention: no workspace"); return CATCOC_E_BAD_ARG; }
  Hq = d.Hq;
  Sq = d.Sq;
  window::WindowParams p;
  memset(&p, 0, sizeof(p));
  const CUtensorMapDataType dt = fmt == CATCOC_FMT_F16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16;
  int rc = encode_bsd(&p.tm_q, q, dt, static_cast<int64_t>(B) * Hq, Sq, D);
  if (rc == 0) rc = encode_bsd(&p.tm_k, k, dt, static_cast<int64_t>(B) * Hk, Sk, D);
  if (rc == 0) rc = encode_bsd(&p.tm_v, v, dt, static_cast<int64_t>(B) * Hk, Sk, D);
  const int64_t rows = static_cast<int64_t>(B) * Hq * Sq, works = static_cast<int64_t>(B) * Hq * d.tiles;
  if (works > (1 << 30)) { set_error("flash_attention: too many query tiles"); return CATCOC_E_TOO_LARGE; }
  if (rc == 0) rc = encode_rows(&p.tm_o, out, dt, static_cast<int64_t>(B) * Hq, Sq, D, 32);
  if (rc != 0) return rc;
  p.part_o = static_cast<float*>(workspace);
  p.part_ml = workspace != nullptr ? p.part_o + d.slices * rows * D : nullptr;
  p.B = B; p.Hq = Hq; p.Hk = Hk; p.Sq = Sq; p.Sk = Sk; p.pos = pos;
  p.window = window; p.sinks = sinks;
  p.tiles = d.tiles; p.works = static_cast<int>(works); p.slices = d.slices; p.per = d.per;
  p.by_works.set(static_cast<uint32_t>(works));
  p.by_heads.set(static_cast<uint32_t>(B) * Hq);
  p.by_hq.set(static_cast<uint32_t>(Hq));
  p.by_group.set(static_cast<uint32_t>(Hq / Hk));
  p.by_pos.set(static_cast<uint32_t>(pos));
  p.scale_log2 = scale * 1.4426950408889634f;
  const uint32_t f = fmt == CATCOC_FMT_BF16 ? 1u : 0u;
  p.idesc_qk = ptx::make_instr_desc(1u, f, f, 0u, 0u, 128u, 128u);
  p.idesc_pv = ptx::make_instr_desc(1u, f, f, 0u, 1u, 128u, static_cast<uint32_t>(D));
  p.status = status;
  p.timeout_ns = timeout_ns ? timeout_ns : 10000000000ull;
  cudaStream_t stream = static_cast<cudaStream_t>(stream_);
  const dim3 grid(static_cast<unsigned>(std::min<int64_t>(works * d.slices, sms)));
  const int db = D / 64, slots = D == 128 ? 4 : 8;
  const size_t smem = static_cast<size_t>(window::kTiles * db + slots * db) * window::kBlockBytes + window::kOutBytes + sizeof(window::Bars) + 1024;
  auto launch = [&](auto kernel) -> int {
    CATCOC_CUDA_OK(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(smem)));
    CATCOC_CUDA_OK(launch_overlapped(kernel, grid, dim3(window::kThreads), smem, stream, p));
    return CATCOC_OK;
  };
  auto call = [&](auto dim, auto type) -> int {
    constexpr int kD = decltype(dim)::value, kF = decltype(type)::value;
    if (d.slices == 1) return launch(window::window_attn_kernel<kD, kF, false>);
    const int first = launch(window::window_attn_kernel<kD, kF, true>);
    if (first != CATCOC_OK) return first;
    CATCOC_CUDA_OK(launch_overlapped(attn::flash_slices_kernel<kD, kF>, dim3(static_cast<unsigned>((rows + 3) / 4)), dim3(128), 0, stream, p.part_o, p.part_ml,
                                     out, rows, d.slices));
    return CATCOC_OK;
  };
  using F16 = std::integral_constant<int, FMT_F16>;
  using BF16 = std::integral_constant<int, FMT_BF16>;
  if (D == 128) return fmt == CATCOC_FMT_BF16 ? call(std::integral_constant<int, 128>{}, BF16{}) : call(std::integral_constant<int, 128>{}, F16{});
  return fmt == CATCOC_FMT_BF16 ? call(std::integral_constant<int, 64>{}, BF16{}) : call(std::integral_constant<int, 64>{}, F16{});
}
