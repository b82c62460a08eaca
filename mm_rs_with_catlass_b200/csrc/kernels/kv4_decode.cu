// Attention of a decode step over the paged 4-bit cache (layout: catcoc/kv4.h).
//
// The query heads that share a KV head, and the new tokens of a sequence, are the rows of a unit (up to 16 of them); every code is read
// once for all of them. The blocks of all units form one list, by the lengths on the device, that is cut into equal runs over the CTAs;
// pieces of a unit that lies in several runs are merged by a second kernel, and a third one adds the probabilities to the caller's sums.
//
//   warps 0..3  a quarter of a stage's tokens each (four blocks, or two), with a softmax and an O of their own; merged at the end of a unit
//   warp 4      producer: walks the run; what the next part is and its rows of q, and one bulk copy a block (72 D bytes) into a ring of stages
//
// Both products run on codes, without their values: with scales and zeros constant over a group g of channels,
//   q . k_j = sum_g s_jg (sum_c q_c code_jc) + z_jg (sum_c q_c),   o_c = sum_j (p_j s_jg) code_jc + sum_j p_j z_jg,
// so that a code costs a mask (five instructions for eight codes of K, six for V's): four bits at the bottom of a half are the subnormal
// code * 2^-24, those above them code * 2^-20, both exact operands. The 16 between them goes into q and into the result. q is brought into
// the range of a half by a power of two per row, p s by one per group that follows the largest scale, so that the only rounding in
// front of the accumulators is that of p s to 11 bits. For that rounding V's codes count from 8, o_c = sum_j (p_j s_jg) (code_jc - 8) +
// sum_j p_j (z_jg + 8 s_jg), with 8 times the sum of the rounded p s taken off at the end (one product with ones a tile): counted from 0 it would
// come multiplied by codes twice as large as the values, 6.2e-4 of an fp16 output where 2.4e-4 remain.
//
// S^T = K q^T has the tokens as rows of mma.m16n8k16; its accumulator, scaled, rounded and transposed by movmatrix, is the second operand of
// O^T += V^T (p s). With up to four rows over two groups of channels (PAIR) the eight columns are four rows of each group, so that no lane
// works on columns that do not exist.
//
// Bound by instruction issue. The products are a stream of codes that have to become 16-bit operands, 43 a cycle and SM at the memory's rate;
// in the registers they are operands as soon as they are masked. The tensor cores' own memory was built too and was slower (16 x 8 heads x
// 4096 tokens, four rows, 75 MB): K into TMEM and V into shared memory as halves, scores a token a thread, tcgen05.mma for both products took
// 37.6 us with four warps twice on an SM and 38.5 us with four teams of four warps and a fifth for issue and copies: a step of 128 tokens was a
// chain of eight waits of 500 to 1900 cycles.
#include <cuda_fp16.h>
#include <algorithm>
#include <cstring>
#include <type_traits>

#include "catcoc/capi.h"
#include "catcoc/host_util.h"
#include "catcoc/kv4.h"
#include "catcoc/params.h"
#include "catcoc/ptx.cuh"
#include "catcoc/softmax_row.cuh"

namespace catcoc {
namespace kv4 {

constexpr int kWarps = 4;                          // consumer warps
constexpr int kThreads = 32 * (kWarps + 1), kWorkers = 32 * kWarps;
constexpr int kTile = 16;                          // tokens of a matrix instruction
constexpr int kTilesBlock = kPage / kTile;
constexpr int kPair = 2;                           // blocks that a run is a multiple of
constexpr int kPShift = 5;                         // p s is held times 2^(5 - e), e: exponent of the largest scale; p <= 2^8, so below 2^14

struct DecodeParams {
  const void* q;                 // [B * q_len, Hq, D]
  const uint8_t* cache;
  const int *table, *lens;
  void* out;                     // [B * q_len, Hq, D]
  float* part_o;                 // [cta + unit][rows of a unit][D]
  float* part_ml;                // [cta + unit][rows of a unit][2]
  int* prefix;                   // [B + 1] blocks of a head of all sequences before
  float* row_ml;                 // [B * Hk][R][2], with weights
  float* scores;                 // [B * Hk][R][S], with weights
  int B, q_len, Hq, Hk, group, R, chunks, max_pages, pages, S;
  int window, sinks;             // window 0: none
  float scale_log2;
  uint32_t* status;
  uint64_t timeout_ns;
};

CATCOC_DEVICE bool sees(int pos, int key, int window, int sinks) {
  return key <= pos && (window == 0 || pos - key < window || key < sinks);
}

// Blocks of a sequence that a row of it may see: the first `sink` ones and [first, last)
struct Span {
  int sink, first, last;
  CATCOC_DEVICE int count() const { return sink + last - first; }
  CATCOC_DEVICE int block(int i) const { return i < sink ? i : first + i - sink; }
};
CATCOC_DEVICE Span span_of(int len, int q_len, int window, int sinks) {
  Span s{0, 0, (len + kPage - 1) / kPage};
  if (window > 0) {
    const int lo = len - q_len - window + 1;       // first key of the first new token's window
    s.first = lo > 0 ? lo / kPage : 0;
    s.sink = min((sinks + kPage - 1) / kPage, s.first);
  }
  return s;
}

// The list in runs, one a CTA: pairs of blocks, as many each and one more in the first ones (whose SMs are different ones), or single blocks
// while there are no more of them than CTAs. Run c begins at run_begin(c); block x is in run run_of(x).
CATCOC_DEVICE int run_begin(int c, int total, int ctas) {
  if (total <= ctas) return min(c, total);
  const int pairs = (total + kPair - 1) / kPair, each = pairs / ctas;
  return min(total, kPair * (c * each + min(c, pairs - each * ctas)));
}
CATCOC_DEVICE int run_of(int x, int total, int ctas) {
  if (total <= ctas) return x;
  const int pairs = (total + kPair - 1) / kPair, each = pairs / ctas, more = pairs - each * ctas, y = x / kPair;
  return y < more * (each + 1) ? y / (each + 1) : more + (y - more * (each + 1)) / each;   // (each is 0 only where all pairs are in the first runs)
}

CATCOC_DEVICE void mma_f16(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
               : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
               : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
CATCOC_DEVICE uint32_t transpose8(uint32_t x) {
  uint32_t y;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}
CATCOC_DEVICE uint32_t half2_of(float lo, float hi) {
  const __half2 h = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&h);
}

CATCOC_DEVICE bool vote_any(bool pred) {           // of the consumer warps
  uint32_t r;
  asm volatile("{\n\t.reg .pred p, q;\n\tsetp.ne.u32 p, %1, 0;\n\tbarrier.cta.red.or.pred q, 1, %2, p;\n\tselp.u32 %0, 1, 0, q;\n\t}\n"
               : "=r"(r) : "r"(static_cast<uint32_t>(pred)), "n"(kWorkers) : "memory");
  return r != 0u;
}

// Row of a matrix instruction -> token of the tile. Two tokens of a pair are swapped in every other pair, so that the rows that four
// lanes read of V lie in both halves of the banks (K's stay free of conflicts).
CATCOC_DEVICE int token_of(int row) { return row ^ ((row >> 1) & 1); }

// A part of the run: blocks [i0, i1) of the n of a unit's list. The sequence's units (Hk x chunks of n blocks) begin at `base` of the list.
struct Part {
  int b, base, n, len;
  int unit, i0, i1;
};

// NT: rows of a unit in eights; PAIR: four rows (D = 128)
template <int D, int NT, bool PAIR>
struct Geo {
  static constexpr int G = Block<D>::kGroups;
  static constexpr int kRows = PAIR ? 4 : 8 * NT;
  // Tiles at once, blocks of a stage, CTAs of an SM: with few rows the chains of a tile (product, exp2, rounding, transpose, product) leave
  // most issue slots empty, and four tiles at once in two CTAs of 168 registers pass two at once in three of 128: 16 x 8 heads x 4096 tokens,
  // four rows, 27.2 -> 25.9 us (one at once in four of 96: 30.0), eight rows, two tiles, 29.2 -> 27.9, D = 64 20.0 -> 18.9.
  static constexpr int kTiles = NT == 2 ? 1 : PAIR || G == 1 ? 4 : 2;
  static constexpr int kSub = NT == 2 ? 2 : 4;     // blocks of a stage
  static constexpr int kStages = NT == 2 ? 3 : 2;
  static constexpr int kCtas = 2;                  // of an SM
};
template <int D, int NT, bool PAIR>
struct Smem {
  using Ge = Geo<D, NT, PAIR>;
  alignas(16) uint8_t stage[Ge::kStages][Ge::kSub][Block<D>::kBytes];
  float o[kWarps][Ge::kRows][D + 4];   // (4: the lanes of a warp store to different banks)
  float2 ml[kWarps][Ge::kRows];
  alignas(16) uint16_t q[2][Ge::kRows * D];   // the rows of a part, and of the one behind it
  Part part[2];                        // n = 0: the run is at its end
  uint32_t there[Ge::kStages];         // which of a stage's blocks are in the cache, a bit each
  uint64_t full[Ge::kStages], empty[Ge::kStages], part_full[2], part_empty[2];
  uint32_t abort_flag, failed[kWarps];
};
static_assert(2 * (sizeof(Smem<128, 2, false>) + 1024) <= 228 * 1024 && 2 * (sizeof(Smem<128, 1, false>) + 1024) <= 228 * 1024, "the CTAs of an SM share its memory");

// D: head dimension, FMT: type of q and out, W: the scores are written for the weights
template <int D, int FMT, int NT, bool PAIR, bool W>
__global__ void __launch_bounds__(kThreads, Geo<D, NT, PAIR>::kCtas) kv4_decode_kernel(const __grid_constant__ DecodeParams p) {
  using L = Block<D>;
  using Ge = Geo<D, NT, PAIR>;
  using Sm = Smem<D, NT, PAIR>;
  static_assert(!PAIR || (NT == 1 && L::kGroups == 2));
  constexpr int G = Ge::G, kRows = Ge::kRows, kSub = Ge::kSub;
  constexpr int GL = PAIR ? 1 : G;               // groups of channels that a lane's columns stand for
  extern __shared__ __align__(16) uint8_t smem_raw[];
  Sm& sm = *reinterpret_cast<Sm*>(smem_raw);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  volatile uint32_t* abort_flag = &sm.abort_flag;
  const int per_seq = p.Hk * p.chunks;            // units of a sequence
  auto span_at = [&](int len) { return span_of(len, p.q_len, p.window, p.sinks); };

  if (threadIdx.x == 0) {
    for (int s = 0; s < Ge::kStages; ++s) { ptx::mbar_init(&sm.full[s], 1); ptx::mbar_init(&sm.empty[s], kWarps); }
    for (int s = 0; s < 2; ++s) { ptx::mbar_init(&sm.part_full[s], 1); ptx::mbar_init(&sm.part_empty[s], kWarps); }
    sm.abort_flag = 0;
    ptx::mbar_fence_init();
  }
  __syncthreads();
  ptx::grid_dependency_wait();
  ptx::launch_dependents();
  uint32_t step = 0, parts = 0;                   // stages and parts so far

  if (warp == kWarps) {
    // ------------------------------ producer ------------------------------
    // the blocks of all sequences, and the sequence in which this CTA's run begins
    int sum = 0;
    for (int b = lane; b < p.B; b += 32) sum += span_at(seq_len(p.lens, b, p.max_pages * kPage, p.status)).count();
    const int total = __reduce_add_sync(0xffffffffu, sum) * per_seq;
    const int begin = run_begin(blockIdx.x, total, static_cast<int>(gridDim.x));
    int behind = 0;
    Part part{0, 0, 0, 0, 0, 0, 0};
    for (int chunk = 0; chunk < p.B; chunk += 32) {
      const int b = chunk + lane, len = b < p.B ? seq_len(p.lens, b, p.max_pages * kPage, p.status) : 0, mine = span_at(len).count();
      int n = mine;
#pragma unroll
      for (int o = 1; o < 32; o *= 2) {
        const int y = __shfl_up_sync(0xffffffffu, n, o);
        if (lane >= o) n += y;
      }
      n += behind;
      if (blockIdx.x == 0 && b < p.B) p.prefix[b + 1] = n;
      const uint32_t hit = __ballot_sync(0xffffffffu, (n - mine) * per_seq <= begin && begin < n * per_seq);
      if (hit != 0u) {
        const int from = __ffs(hit) - 1;
        part.b = chunk + from;
        part.base = __shfl_sync(0xffffffffu, (n - mine) * per_seq, from);
        part.n = __shfl_sync(0xffffffffu, mine, from);
        part.len = __shfl_sync(0xffffffffu, len, from);
        if (blockIdx.x != 0) break;
      }
      behind = __shfl_sync(0xffffffffu, n, 31);
    }
    if (blockIdx.x == 0 && lane == 0) p.prefix[0] = 0;
    const int end = run_begin(blockIdx.x + 1, total, static_cast<int>(gridDim.x));
    // the part of the run that begins at list position `at`, in the sequence of `s` or behind it
    auto settle = [&](Part& s, int at) {
      while (s.base + s.n * per_seq <= at) {
        s.base += s.n * per_seq;
        ++s.b;
        s.len = seq_len(p.lens, s.b, p.max_pages * kPage, p.status);
        s.n = span_at(s.len).count();
      }
      s.unit = (at - s.base) / s.n;
      s.i0 = at - s.base - s.unit * s.n;
      s.i1 = min(s.n, s.i0 + end - at);
    };
    // names of 32 blocks from block i on, as the table has them
    auto names = [&](const Part& s, int i) { return i + lane < s.i1 ? p.table[static_cast<int64_t>(s.b) * p.max_pages + span_at(s.len).block(i + lane)] : 0; };
    int raw = 0;
    if (begin < end) {
      settle(part, begin);
      raw = names(part, part.i0);
    }
    bool ok = true;
    for (int at = begin; ok && at < end; ++parts) {
      const int hk = part.unit / p.chunks, row0 = (part.unit - hk * p.chunks) * kRows, rows = min(kRows, p.R - row0);
      // what the part is, and its rows of q: those of a new token are consecutive heads
      const uint32_t place = parts & 1u;
      ok = ptx::mbar_wait(&sm.part_empty[place], ((parts >> 1) & 1u) ^ 1u, p.timeout_ns, abort_flag);
      if (!ok) break;
      if (lane == 0) {
        sm.part[place] = part;
        ptx::mbar_expect_tx(&sm.part_full[place], static_cast<uint32_t>(rows * D * 2));
        for (int r = row0; r < row0 + rows;) {
          const int tok = r / p.group, next = min(row0 + rows, (tok + 1) * p.group);
          ptx::bulk_load_1d(sm.q[place] + (r - row0) * D,
                            static_cast<const uint16_t*>(p.q) + ((static_cast<int64_t>(part.b) * p.q_len + tok) * p.Hq + hk * p.group + (r - tok * p.group)) * D,
                            static_cast<uint32_t>((next - r) * D * 2), &sm.part_full[place]);
          r = next;
        }
      }
      __syncwarp();
      at += part.i1 - part.i0;
      Part next = part;
      int ids = -1, next_raw = 0;
      uint32_t named = 0;
      for (int i = part.i0; i < part.i1; i += kSub, ++step) {
        const int k = (i - part.i0) & 31;
        // the names of 32 blocks at a time, so that no copy waits for its own (one that is not in the cache is noted, and left out by the consumers)
        if (k == 0) {
          if (i > part.i0) raw = names(part, i);
          ids = i + lane < part.i1 ? checked_page(raw, p.pages, p.status) : -1;
          named = __ballot_sync(0xffffffffu, ids >= 0);
        }
        const uint32_t stage = step % Ge::kStages;
        ok = ptx::mbar_wait(&sm.empty[stage], ((step / Ge::kStages) & 1u) ^ 1u, p.timeout_ns, abort_flag);
        if (!ok) break;
        int page[kSub], found = 0;
#pragma unroll
        for (int s = 0; s < kSub; ++s) {
          page[s] = __shfl_sync(0xffffffffu, ids, k + s);
          found += page[s] >= 0;
        }
        if (lane == 0) {
          sm.there[stage] = named >> k;
          if (found == 0) ptx::mbar_arrive(&sm.full[stage]);
          else ptx::mbar_expect_tx(&sm.full[stage], static_cast<uint32_t>(found * L::kBytes));
#pragma unroll
          for (int s = 0; s < kSub; ++s)
            if (page[s] >= 0)
              ptx::bulk_load_1d(sm.stage[stage][s], p.cache + (static_cast<int64_t>(page[s]) * p.Hk + hk) * L::kBytes, L::kBytes, &sm.full[stage]);
        }
        __syncwarp();
        // (behind the first copies: the next part and its names, under way while this one's are used)
        if (i == part.i0 && at < end) {
          settle(next, at);
          next_raw = names(next, next.i0);
        }
      }
      part = next;
      raw = next_raw;
    }
    if (ok) ok = ptx::mbar_wait(&sm.part_empty[parts & 1u], ((parts >> 1) & 1u) ^ 1u, p.timeout_ns, abort_flag);
    if (ok && lane == 0) {
      sm.part[parts & 1u].n = 0;
      ptx::mbar_arrive(&sm.part_full[parts & 1u]);
    }
    if (!ok || *abort_flag != 0) {
      // the run was given up: the copies that are still on their way land before the block's memory is handed on
      if (lane == 0) *abort_flag = 1;
      volatile uint32_t never = 0;
      for (uint32_t i = step > Ge::kStages ? step - Ge::kStages : 0; i < step; ++i)
        ptx::mbar_wait(&sm.full[i % Ge::kStages], (i / Ge::kStages) & 1u, 100000000ull, &never);
      for (uint32_t i = parts > 2u ? parts - 2u : 0u; i < parts; ++i) ptx::mbar_wait(&sm.part_full[i & 1u], (i >> 1) & 1u, 100000000ull, &never);
    }
    return;
  }

  // ------------------------------ products and softmax ------------------------------
  const int g8 = lane >> 2, t4 = lane & 3;
  const int own = PAIR ? t4 >> 1 : 0;             // PAIR: the group of this lane's columns
  auto row_of = [&](int nt, int c) { return PAIR ? 2 * (t4 & 1) + c : nt * 8 + 2 * t4 + c; };   // row of the unit that a lane's column stands for
  bool ok = true;
  for (;; ++parts) {
    // (every warp takes all barriers of all parts, also after a failed wait; all leave together. The vote is also the barrier behind which
    // the merge's memory is written again.)
    const uint32_t place = parts & 1u;
    ok = ptx::mbar_wait(&sm.part_full[place], (parts >> 1) & 1u, p.timeout_ns, abort_flag);
    if (!ok && lane == 0) *abort_flag = 1;
    ok = !vote_any(!ok);
    if (!ok) break;
    const Part part = sm.part[place];
    if (part.n == 0) break;
    const int b = part.b, len = part.len;
    const Span span = span_at(len);
    const int hk = part.unit / p.chunks, row0 = (part.unit - hk * p.chunks) * kRows;   // first row of the unit among the R of its head
    // q as the second operand of S^T: column g8 of every eight, the channels of this lane's words; b0, b1 of every step
    uint32_t qf[NT][2 * G][4];
    float qscale[NT][2], qsum[NT][GL][2];             // of the rows of this lane's columns: score = qscale * raw score
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      const int row = PAIR ? g8 & 3 : nt * 8 + g8;
      const uint16_t* src = sm.q[place] + row * D;
      float x[2 * G][8], mx = 0.0f, sum[G] = {};
#pragma unroll
      for (int i = 0; i < 2 * G; ++i) {
        uint4 raw = make_uint4(0, 0, 0, 0);
        if (row0 + row < p.R) raw = *reinterpret_cast<const uint4*>(src + (i % G) * 64 + (2 * t4 + i / G) * 8);
        const uint32_t u[4] = {raw.x, raw.y, raw.z, raw.w};
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          if constexpr (FMT == FMT_BF16) { x[i][2 * e] = bf16_lo(u[e]); x[i][2 * e + 1] = bf16_hi(u[e]); }
          else { const float2 v = __half22float2(*reinterpret_cast<const __half2*>(&u[e])); x[i][2 * e] = v.x; x[i][2 * e + 1] = v.y; }
        }
#pragma unroll
        for (int e = 0; e < 8; ++e) { mx = fmaxf(mx, fabsf(x[i][e])); sum[i % G] += x[i][e]; }
      }
      mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
      mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
      // 2^(14 - exponent): the largest element lands in [2^14, 2^15)
      const int ef = min(254, max(1, 268 - static_cast<int>(__float_as_uint(mx) >> 23)));
      const float f = mx > 0.0f ? __uint_as_float(static_cast<uint32_t>(ef) << 23) : 1.0f;
#pragma unroll
      for (int i = 0; i < 2 * G; ++i) {
        // steps of a word: its bits 0-3, 4-7 (and 16-19, 20-23), then 8-11, 12-15 (and 24-27, 28-31)
        const float h = PAIR && i % G != (g8 >> 2) ? 0.0f : f, h16 = h * 0.0625f;   // PAIR: a column knows the channels of its group alone
        qf[nt][i][0] = half2_of(x[i][0] * h, x[i][4] * h);
        qf[nt][i][1] = half2_of(x[i][1] * h16, x[i][5] * h16);
        qf[nt][i][2] = half2_of(x[i][2] * h, x[i][6] * h);
        qf[nt][i][3] = half2_of(x[i][3] * h16, x[i][7] * h16);
      }
      const float back = p.scale_log2 * 16777216.0f / f;
#pragma unroll
      for (int g = 0; g < G; ++g) {
        sum[g] += __shfl_xor_sync(0xffffffffu, sum[g], 1);
        sum[g] += __shfl_xor_sync(0xffffffffu, sum[g], 2);
        sum[g] *= f * (1.0f / 16777216.0f);           // in the unit of the products of codes
      }
      if constexpr (PAIR) sum[0] = g8 < 4 ? sum[0] : sum[1];
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        const int from = (2 * t4 + c) * 4;            // a lane of that column
        qscale[nt][c] = __shfl_sync(0xffffffffu, back, from);
#pragma unroll
        for (int g = 0; g < GL; ++g) qsum[nt][g][c] = __shfl_sync(0xffffffffu, sum[g], from);
      }
    }
    __syncwarp();
    if (lane == 0) ptx::mbar_arrive(&sm.part_empty[place]);
    // m: largest raw score, as far as it is followed; m_neg: minus its score; limit: raw score from which on it moves
    float o[NT][G][4][4] = {}, wsum[NT][GL][4] = {}, m[NT][2], m_neg[NT][2], limit[NT][2], l[NT][2] = {}, zsum[NT][GL][2] = {};
    uint32_t e_ref[GL];                               // exponent field that the scales of V are held against
    float vscale[GL];                                 // 2^(kPShift + 127 - e_ref)
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int c = 0; c < 2; ++c) { m[nt][c] = limit[nt][c] = -INFINITY; m_neg[nt][c] = 0.0f; }
#pragma unroll
    for (int g = 0; g < GL; ++g) { e_ref[g] = 8; vscale[g] = __uint_as_float((254u + kPShift - 8u) << 23); }
    const int pos_lo = len - p.q_len, pos_hi = len - 1;

    // TILES tiles from token `t0` of a block on. ALL: every row sees every key of them.
    auto tiles = [&](auto all_c, auto count_c, const uint8_t* block, int t0, int key0) {
      constexpr bool ALL = decltype(all_c)::value;
      constexpr int TILES = decltype(count_c)::value;
      const uint8_t *kc = block + t0 * L::kRow, *vc = kc + L::kHalf, *kp = block + L::kPar + t0 * L::kParRow, *vp = kp + L::kHalf;
      float s[TILES][NT][4];
      uint32_t vpar[TILES][2][GL];
      const int tk = token_of(g8);
#pragma unroll
      for (int i = 0; i < TILES; ++i) {
        // S^T: rows g8 and g8 + 8 are tokens, channels by t4
        uint32_t ka[2 * G], kb[2 * G], par[2][GL];
        const uint8_t* from = kc + (i * kTile + tk) * L::kRow + t4 * 8 * G;
        if constexpr (G == 2) {
          const uint4 x = *reinterpret_cast<const uint4*>(from), y = *reinterpret_cast<const uint4*>(from + 8 * L::kRow);
          ka[0] = x.x; ka[1] = x.y; ka[2] = x.z; ka[3] = x.w;
          kb[0] = y.x; kb[1] = y.y; kb[2] = y.z; kb[3] = y.w;
        } else {
          const uint2 x = *reinterpret_cast<const uint2*>(from), y = *reinterpret_cast<const uint2*>(from + 8 * L::kRow);
          ka[0] = x.x; ka[1] = x.y;
          kb[0] = y.x; kb[1] = y.y;
        }
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          const int off = (i * kTile + tk + 8 * u) * L::kParRow + own * 4;
          if constexpr (GL == 2) {
            const uint2 x = *reinterpret_cast<const uint2*>(kp + off), y = *reinterpret_cast<const uint2*>(vp + off);
            par[u][0] = x.x; par[u][1] = x.y; vpar[i][u][0] = y.x; vpar[i][u][1] = y.y;
          } else {
            par[u][0] = *reinterpret_cast<const uint32_t*>(kp + off); vpar[i][u][0] = *reinterpret_cast<const uint32_t*>(vp + off);
          }
        }
        float acc[NT][G][4] = {};                     // (PAIR: the groups' columns differ, their sum is both)
#pragma unroll
        for (int w = 0; w < 2 * G; ++w) {
          const uint32_t a8 = ka[w] >> 8, b8 = kb[w] >> 8;
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) {
            mma_f16(acc[nt][w % G], ka[w] & 0x000f000fu, kb[w] & 0x000f000fu, ka[w] & 0x00f000f0u, kb[w] & 0x00f000f0u, qf[nt][w][0], qf[nt][w][1]);
            mma_f16(acc[nt][w % G], a8 & 0x000f000fu, b8 & 0x000f000fu, a8 & 0x00f000f0u, b8 & 0x00f000f0u, qf[nt][w][2], qf[nt][w][3]);
          }
        }
        // raw scores of tokens g8 ([0], [1]) and g8 + 8 ([2], [3]), this lane's two columns
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const int u = e >> 1, c = e & 1;
            float a = bf16_hi(par[u][0]) * qsum[nt][0][c];
            if constexpr (PAIR) {
              a = fmaf(bf16_lo(par[u][0]), acc[nt][0][e] + acc[nt][G - 1][e], a);
              a += __shfl_xor_sync(0xffffffffu, a, 2);
            } else {
#pragma unroll
              for (int g = 1; g < G; ++g) a = fmaf(bf16_hi(par[u][g]), qsum[nt][g][c], a);
#pragma unroll
              for (int g = 0; g < G; ++g) a = fmaf(bf16_lo(par[u][g]), acc[nt][g][e], a);
            }
            s[i][nt][e] = a;
          }
        if constexpr (!ALL) {
          // what a row does not see weighs nothing, whatever the cache holds there
          bool seen[2] = {false, false};
#pragma unroll
          for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const int r = row0 + row_of(nt, e & 1);
              const bool v = r < p.R && sees(pos_lo + r / p.group, key0 + i * kTile + tk + 8 * (e >> 1), p.window, p.sinks);
              if (!v) s[i][nt][e] = -INFINITY;
              seen[e >> 1] |= v;
            }
#pragma unroll
          for (int u = 0; u < 2; ++u)
#pragma unroll
            for (int g = 0; g < GL; ++g)
              if (!seen[u]) vpar[i][u][g] = 0u;
        }
        if constexpr (W) {
          float* dst = p.scores + (static_cast<int64_t>(b) * p.Hk + hk) * p.R * p.S + key0 + i * kTile + tk;
#pragma unroll
          for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int c = 0; c < 2; ++c) {
              const int r = row0 + row_of(nt, c);
              if (r < p.R && own == 0) {
                dst[static_cast<int64_t>(r) * p.S] = s[i][nt][c] * qscale[nt][c];
                dst[static_cast<int64_t>(r) * p.S + 8] = s[i][nt][2 + c] * qscale[nt][c];
              }
            }
        }
      }
      // the references: m moves when a score exceeds its own by more than 8, e_ref when a scale is past twice its power
      float ps[TILES][GL][2], top = 0.0f;
#pragma unroll
      for (int i = 0; i < TILES; ++i)
#pragma unroll
        for (int g = 0; g < GL; ++g)
#pragma unroll
          for (int u = 0; u < 2; ++u) {
            ps[i][g][u] = bf16_lo(vpar[i][u][g]) * vscale[g];
            top = fmaxf(top, ps[i][g][u]);
          }
      bool move = top >= static_cast<float>(2 << kPShift);
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          float x = fmaxf(s[0][nt][c], s[0][nt][2 + c]);
#pragma unroll
          for (int i = 1; i < TILES; ++i) x = ptx::max3(x, s[i][nt][c], s[i][nt][2 + c]);
          move |= x > limit[nt][c];
        }
      if (__any_sync(0xffffffffu, move)) {
        float beta[GL];
#pragma unroll
        for (int g = 0; g < GL; ++g) {
          // (scales are not negative; one that is no number, or infinite, sets no reference)
          uint32_t e_new = e_ref[g];
#pragma unroll
          for (int i = 0; i < TILES; ++i)
#pragma unroll
            for (int u = 0; u < 2; ++u) {
              const uint32_t x = (vpar[i][u][g] >> 7) & 0xffu;
              e_new = max(e_new, x == 255u ? 0u : x);
            }
#pragma unroll
          for (int d = 1; d < 32; d *= 2)
            if (d != 2) e_new = max(e_new, __shfl_xor_sync(0xffffffffu, e_new, d));   // (lanes t4 and t4 ^ 2 may stand for two groups)
          beta[g] = e_new - e_ref[g] > 126u ? 0.0f : __uint_as_float((127u + e_ref[g] - e_new) << 23);
          e_ref[g] = e_new;
          vscale[g] = __uint_as_float((254u + kPShift - e_new) << 23);
#pragma unroll
          for (int i = 0; i < TILES; ++i)
#pragma unroll
            for (int u = 0; u < 2; ++u) ps[i][g][u] = bf16_lo(vpar[i][u][g]) * vscale[g];
        }
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int c = 0; c < 2; ++c) {
            float x = fmaxf(s[0][nt][c], s[0][nt][2 + c]);
#pragma unroll
            for (int i = 1; i < TILES; ++i) x = ptx::max3(x, s[i][nt][c], s[i][nt][2 + c]);
#pragma unroll
            for (int d = 4; d < 32; d *= 2) x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, d));
            const float mn = fmaxf(m[nt][c], x), neg = mn == -INFINITY ? 0.0f : -mn * qscale[nt][c];
            const float alpha = m[nt][c] == -INFINITY ? 0.0f : ptx::ex2_approx(neg - m_neg[nt][c]);
            m[nt][c] = mn;
            m_neg[nt][c] = neg;
            limit[nt][c] = mn + attn::kLazyRescale / qscale[nt][c];
            l[nt][c] *= alpha;
#pragma unroll
            for (int g = 0; g < GL; ++g) {
              zsum[nt][g][c] *= alpha;
              wsum[nt][g][c] *= alpha * beta[g];
            }
#pragma unroll
            for (int g = 0; g < G; ++g)
#pragma unroll
              for (int k = 0; k < 4; ++k) {
                o[nt][g][k][c] *= alpha * beta[g % GL];
                o[nt][g][k][2 + c] *= alpha * beta[g % GL];
              }
          }
      }
#pragma unroll
      for (int i = 0; i < TILES; ++i) {
        uint32_t pb[NT][GL][2];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
          float pr[4];
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            pr[e] = ptx::ex2_approx(fmaf(s[i][nt][e], qscale[nt][e & 1], m_neg[nt][e & 1]));
            l[nt][e & 1] += pr[e];
          }
#pragma unroll
          for (int g = 0; g < GL; ++g) {
            float w[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              w[e] = pr[e] * ps[i][g][e >> 1];
              float z = fmaf(8.0f, bf16_lo(vpar[i][e >> 1][g]), bf16_hi(vpar[i][e >> 1][g]));
              if (!ALL && s[i][nt][e] == -INFINITY) { w[e] = 0.0f; z = 0.0f; }
              zsum[nt][g][e & 1] = fmaf(pr[e], z, zsum[nt][g][e & 1]);
            }
            pb[nt][g][0] = transpose8(half2_of(w[0], w[1]));
            pb[nt][g][1] = transpose8(half2_of(w[2], w[3]));
            mma_f16(wsum[nt][g], 0x3c003c00u, 0x3c003c00u, 0x3c003c00u, 0x3c003c00u, pb[nt][g][0], pb[nt][g][1]);
          }
        }
        // O^T: rows g8 and g8 + 8 are the channels 64 g + 8 g8 + 2 k and + 1, tokens of the rows 2 t4, 2 t4 + 1, + 8, + 9
        uint32_t vw[4][G];
#pragma unroll
        for (int u = 0; u < 4; ++u) {
          const uint8_t* from = vc + (i * kTile + token_of(2 * t4 + (u & 1)) + 8 * (u >> 1)) * L::kRow + g8 * 4 * G;
          if constexpr (G == 2) { const uint2 x = *reinterpret_cast<const uint2*>(from); vw[u][0] = x.x; vw[u][1] = x.y; }
          else vw[u][0] = *reinterpret_cast<const uint32_t*>(from);
        }
#pragma unroll
        for (int g = 0; g < G; ++g)
#pragma unroll
          for (int hw = 0; hw < 2; ++hw) {
            const uint32_t x = __byte_perm(vw[0][g], vw[1][g], hw ? 0x7632 : 0x5410), y = __byte_perm(vw[2][g], vw[3][g], hw ? 0x7632 : 0x5410);
            const uint32_t x8 = x >> 8, y8 = y >> 8;
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
              mma_f16(o[nt][g][2 * hw], x & 0x000f000fu, x & 0x00f000f0u, y & 0x000f000fu, y & 0x00f000f0u, pb[nt][g % GL][0], pb[nt][g % GL][1]);
              mma_f16(o[nt][g][2 * hw + 1], x8 & 0x000f000fu, x8 & 0x00f000f0u, y8 & 0x000f000fu, y8 & 0x00f000f0u, pb[nt][g % GL][0], pb[nt][g % GL][1]);
            }
          }
      }
    };

#pragma unroll 1
    for (int i = part.i0; i < part.i1; i += kSub, ++step) {
      const uint32_t stage = step % Ge::kStages;
      ok = ptx::mbar_wait(&sm.full[stage], (step / Ge::kStages) & 1u, p.timeout_ns, abort_flag);
      if (!ok) break;
      // Tiles that all rows see whole go several at once, as their state fits the registers; the others by themselves
      auto whole = [&](int key0, int n) {
        const int behind = key0 + n * kTile;
        return behind - 1 <= pos_lo && (p.window == 0 || pos_hi - key0 < p.window || behind <= p.sinks);
      };
      auto masked = [&](const uint8_t* block, int t0, int key0) {
        if (key0 <= pos_hi && (p.window == 0 || pos_lo - (key0 + kTile - 1) < p.window || key0 < p.sinks))
          tiles(std::false_type{}, std::integral_constant<int, 1>{}, block, t0, key0);
      };
      // First key of a tile; that of a block that is not in the cache lies behind all that any row sees, and the block is left out
      const uint32_t there = sm.there[stage];
      auto first_key = [&](int at, int t0) { return (there >> at) & 1u ? span.block(i + at) * kPage + t0 : 1 << 30; };
      const int count = min(kSub, part.i1 - i);
      if constexpr (NT == 2) {
        // (half a block a warp)
        const int at = warp / 2, t0 = warp % 2 * 2 * kTile;
        if (at < count) {
          const int key0 = first_key(at, t0);
          const uint8_t* block = sm.stage[stage][at];
          if (whole(key0, 2)) {
#pragma unroll 1
            for (int t = 0; t < 2 * kTile; t += kTile) tiles(std::true_type{}, std::integral_constant<int, 1>{}, block, t0 + t, key0 + t);
          } else {
#pragma unroll 1
            for (int t = 0; t < 2 * kTile; t += kTile) masked(block, t0 + t, key0 + t);
          }
        }
      } else {
        // The tiles of the stage's blocks, as many for each warp. Several go at once only from where they end in their block and in this
        // warp's share: behind the first, masked tiles of a window the walk may stand anywhere. (Both numbers in one test: as two, D = 64 takes
        // 19.9 us instead of 18.6 for 16 x 8 heads x 4096 tokens. A block's two pairs behind one test: 131072 tokens, eight rows, 46.4 -> 45.8.)
        const uint32_t end = (warp + 1) * count;
        for (uint32_t t = warp * count; t < end;) {
          const int at = static_cast<int>(t / kTilesBlock), t0 = static_cast<int>(t % kTilesBlock) * kTile, key0 = first_key(at, t0);
          const uint8_t* block = sm.stage[stage][at];
          const uint32_t most = (t | count) & 3u;
          if (Ge::kTiles == 4 && most == 0u && whole(key0, 4)) {
            tiles(std::true_type{}, std::integral_constant<int, Ge::kTiles>{}, block, t0, key0);
            t += 4u;
          } else if ((most & 1u) == 0u && whole(key0, 2)) {
            const int n = Ge::kTiles == 2 && most == 0u && whole(key0, 4) ? 4 : 2;
#pragma unroll 1
            for (int u = 0; u < n; u += 2) tiles(std::true_type{}, std::integral_constant<int, 2>{}, block, t0 + u * kTile, key0 + u * kTile);
            t += static_cast<uint32_t>(n);
          } else {
            if (whole(key0, 1)) tiles(std::true_type{}, std::integral_constant<int, 1>{}, block, t0, key0);
            else masked(block, t0, key0);
            ++t;
          }
        }
      }
      __syncwarp();
      if (lane == 0) ptx::mbar_arrive(&sm.empty[stage]);
    }

    // the four warps' pieces of the unit: every one leaves its row, weighed against the largest maximum
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int c = 0; c < 2; ++c) {
#pragma unroll
        for (int d = 4; d < 32; d *= 2) {
          l[nt][c] += __shfl_xor_sync(0xffffffffu, l[nt][c], d);
#pragma unroll
          for (int g = 0; g < GL; ++g) zsum[nt][g][c] += __shfl_xor_sync(0xffffffffu, zsum[nt][g][c], d);
        }
        // (from here on m is a score)
        m[nt][c] = m[nt][c] == -INFINITY ? -INFINITY : -m_neg[nt][c];
        if (g8 == 0 && own == 0) sm.ml[warp][row_of(nt, c)] = make_float2(m[nt][c], l[nt][c]);
      }
    if (!ok && lane == 0) *abort_flag = 1;
    if (lane == 0) sm.failed[warp] = ok ? 0u : 1u;
    ptx::named_bar_sync(1, kWorkers);
    ok = (sm.failed[0] | sm.failed[1] | sm.failed[2] | sm.failed[3]) == 0u;
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        const int r = row_of(nt, c);
        float mt = sm.ml[0][r].x;
#pragma unroll
        for (int w = 1; w < kWarps; ++w) mt = fmaxf(mt, sm.ml[w][r].x);
        const float a = m[nt][c] == -INFINITY ? 0.0f : ptx::ex2_approx(m[nt][c] - mt);
#pragma unroll
        for (int g = 0; g < GL; ++g) {
          // 2^24 and 2^(e_ref - 127 - 5) undone in two steps: either alone could leave the range
          const float f1 = __uint_as_float(e_ref[g] << 23), f2 = a * (16777216.0f / (1 << kPShift));
          const float eights = wsum[nt][g][c] * (a * (-8.0f / (1 << kPShift)));
          float4 v[2];
          float* f = reinterpret_cast<float*>(v);
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            // (PAIR: the columns of the other group are of no use)
            const float x = PAIR && own == 1 ? o[nt][G - 1][k][c] : o[nt][g][k][c], y = PAIR && own == 1 ? o[nt][G - 1][k][2 + c] : o[nt][g][k][2 + c];
            f[2 * k] = fmaf(fmaf(x, f2, eights), f1, a * zsum[nt][g][c]);
            f[2 * k + 1] = fmaf(fmaf(y, f2 * 0.0625f, eights), f1, a * zsum[nt][g][c]);
          }
          // (a warp that saw nothing of a row has nothing to add, not zero times what it holds)
          if (m[nt][c] == -INFINITY && l[nt][c] == 0.0f) v[0] = v[1] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
          float4* dst = reinterpret_cast<float4*>(&sm.o[warp][r][(PAIR ? own : g) * 64 + g8 * 8]);
          dst[0] = v[0];
          dst[1] = v[1];
        }
      }
    ptx::named_bar_sync(1, kWorkers);
    if (!ok) break;
    // thread: eight columns of a row
    const bool alone = part.i1 - part.i0 == part.n;
    for (int x = threadIdx.x; x < kRows * (D / 8); x += kWorkers) {
      const int r = x / (D / 8), col = (x % (D / 8)) * 8, rr = row0 + r;
      if (rr >= p.R) continue;
      float mt = -INFINITY, lt = 0.0f, v[8] = {};
#pragma unroll
      for (int w = 0; w < kWarps; ++w) mt = fmaxf(mt, sm.ml[w][r].x);
#pragma unroll
      for (int w = 0; w < kWarps; ++w) {
        const float2 ml = sm.ml[w][r];
        const float wgt = ml.x == -INFINITY ? (ml.y == 0.0f ? 0.0f : 1.0f) : ptx::ex2_approx(ml.x - mt);
        lt += wgt * ml.y;
        const float4 y0 = *reinterpret_cast<const float4*>(&sm.o[w][r][col]), y1 = *reinterpret_cast<const float4*>(&sm.o[w][r][col + 4]);
        v[0] += y0.x; v[1] += y0.y; v[2] += y0.z; v[3] += y0.w;
        v[4] += y1.x; v[5] += y1.y; v[6] += y1.z; v[7] += y1.w;
      }
      if (alone) {
        const float inv = lt == 0.0f ? 0.0f : 1.0f / lt;
        const int tok = rr / p.group;
        uint16_t* dst = static_cast<uint16_t*>(p.out) + ((static_cast<int64_t>(b) * p.q_len + tok) * p.Hq + hk * p.group + (rr - tok * p.group)) * D + col;
        ptx::st_global_v4(dst, make_uint4(attn::pack16<FMT>(v[0] * inv, v[1] * inv), attn::pack16<FMT>(v[2] * inv, v[3] * inv),
                                          attn::pack16<FMT>(v[4] * inv, v[5] * inv), attn::pack16<FMT>(v[6] * inv, v[7] * inv)));
        if (W && col == 0) *reinterpret_cast<float2*>(p.row_ml + ((static_cast<int64_t>(b) * p.Hk + hk) * p.R + rr) * 2) = make_float2(mt, lt);
      } else {
        const int64_t piece = (static_cast<int64_t>(blockIdx.x) + b * per_seq + part.unit) * kRows + r;
        float4* dst = reinterpret_cast<float4*>(p.part_o + piece * D + col);
        dst[0] = make_float4(v[0], v[1], v[2], v[3]);
        dst[1] = make_float4(v[4], v[5], v[6], v[7]);
        if (col == 0) *reinterpret_cast<float2*>(p.part_ml + piece * 2) = make_float2(mt, lt);
      }
    }
  }
  // a wait that ran out of time, noted once for the launch
  if (!ok && threadIdx.x == 0 && atomicCAS(p.status, 0u, static_cast<uint32_t>(STATUS_TIMEOUT_PIPELINE)) == 0u) {
    p.status[1] = 0u; p.status[2] = 400u; p.status[3] = 0u; p.status[4] = 0u; p.status[5] = 0u; p.status[6] = blockIdx.x;
    __threadfence_system();
  }
}

// Merges the pieces of the units that were cut, a warp a row, 32 pieces at a time; rows of sequences without a block are zero.
template <int D, int FMT, bool W>
__global__ void __launch_bounds__(128) kv4_combine_kernel(const DecodeParams p, int rows_unit, int ctas) {
  constexpr int kPer = D / 32;
  ptx::grid_dependency_wait();
  ptx::launch_dependents();
  const int per_seq = p.Hk * p.chunks, unit = blockIdx.x, b = unit / per_seq, in_seq = unit - b * per_seq;
  const int r = blockIdx.y * 4 + (threadIdx.x >> 5), lane = threadIdx.x & 31;
  const int hk = in_seq / p.chunks, rr = (in_seq - hk * p.chunks) * rows_unit + r;
  if (r >= rows_unit || rr >= p.R) return;
  const int n = p.prefix[b + 1] - p.prefix[b], total = p.prefix[p.B] * per_seq;
  const int first = p.prefix[b] * per_seq + in_seq * n;
  const int tok = rr / p.group;
  uint16_t* dst = static_cast<uint16_t*>(p.out) + ((static_cast<int64_t>(b) * p.q_len + tok) * p.Hq + hk * p.group + (rr - tok * p.group)) * D + lane * kPer;
  float m = -INFINITY, l = 0.0f, acc[kPer] = {};
  if (n > 0) {
    const int c0 = run_of(first, total, ctas), c1 = run_of(first + n - 1, total, ctas);
    if (c0 == c1) return;                          // written by its CTA
    for (int base = c0; base <= c1; base += 32) {
      const int count = min(32, c1 + 1 - base);
      const int64_t piece = (static_cast<int64_t>(base) + unit) * rows_unit + r;      // piece c: + c * rows_unit
      const float2 ml = lane < count ? *reinterpret_cast<const float2*>(p.part_ml + (piece + static_cast<int64_t>(lane) * rows_unit) * 2) : make_float2(-INFINITY, 0.0f);
      float mx = fmaxf(m, ml.x);
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, o));
      const float old = m == -INFINITY ? 0.0f : ptx::ex2_approx(m - mx);
      const float w = ml.x == -INFINITY ? (ml.y == 0.0f ? 0.0f : 1.0f) : ptx::ex2_approx(ml.x - mx);
      float wl = w * ml.y;
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) wl += __shfl_xor_sync(0xffffffffu, wl, o);
      m = mx;
      l = l * old + wl;
#pragma unroll
      for (int e = 0; e < kPer; ++e) acc[e] *= old;
#pragma unroll 8
      for (int c = 0; c < count; ++c) {
        const float wc = __shfl_sync(0xffffffffu, w, c);
        const float* src = p.part_o + (piece + static_cast<int64_t>(c) * rows_unit) * D + lane * kPer;
        float o[kPer];
        if constexpr (kPer == 4) *reinterpret_cast<float4*>(o) = *reinterpret_cast<const float4*>(src);
        else *reinterpret_cast<float2*>(o) = *reinterpret_cast<const float2*>(src);
#pragma unroll
        for (int e = 0; e < kPer; ++e) acc[e] += wc * o[e];
      }
    }
  }
  const float inv = l == 0.0f ? 0.0f : 1.0f / l;
#pragma unroll
  for (int e = 0; e < kPer / 2; ++e) reinterpret_cast<uint32_t*>(dst)[e] = attn::pack16<FMT>(acc[2 * e] * inv, acc[2 * e + 1] * inv);
  if (W && lane == 0) *reinterpret_cast<float2*>(p.row_ml + ((static_cast<int64_t>(b) * p.Hk + hk) * p.R + rr) * 2) = make_float2(m, l);
}

// weights[b, hk, j] += sum over the rows of 2^(score - m) / l, in the order of the rows
__global__ void __launch_bounds__(256) kv4_weights_kernel(const DecodeParams p, float* weights, int64_t pitch) {
  extern __shared__ float2 row[];
  ptx::grid_dependency_wait();
  const int bh = blockIdx.x, b = bh / p.Hk;
  const int len = min(max(p.lens[b], 0), p.max_pages * kPage);
  const int j0 = static_cast<int>(blockIdx.z * gridDim.y + blockIdx.y) * 256, j = j0 + threadIdx.x;   // (2^24 tokens are 65536 blocks, one more than grid y has)
  if (j0 >= len) return;
  // (what is not in the cache has no scores)
  const bool there = j < len && static_cast<uint32_t>(p.table[static_cast<int64_t>(b) * p.max_pages + j / kPage]) < static_cast<uint32_t>(p.pages);
  for (int r = threadIdx.x; r < p.R; r += 256) {
    const float2 ml = *reinterpret_cast<const float2*>(p.row_ml + (static_cast<int64_t>(bh) * p.R + r) * 2);
    row[r] = make_float2(ml.x == -INFINITY ? 0.0f : ml.x, ml.y == 0.0f ? 0.0f : 1.0f / ml.y);
  }
  __syncthreads();
  if (!there) return;
  const float* s = p.scores + static_cast<int64_t>(bh) * p.R * p.S + j;
  float sum = 0.0f;
#pragma unroll 4
  for (int r = 0; r < p.R; ++r) {
    const int pos = len - p.q_len + r / p.group;
    if (sees(pos, j, p.window, p.sinks)) sum += ptx::ex2_approx(s[static_cast<int64_t>(r) * p.S] - row[r].x) * row[r].y;
  }
  if (sum != 0.0f) weights[bh * pitch + j] += sum;
}

}  // namespace kv4
}  // namespace catcoc

using namespace catcoc;
using namespace catcoc::host;
using namespace catcoc::kv4;

namespace {
struct DecodePlan {
  int R, rows, chunks;      // rows: of a unit, as the kernel is built for them
  int64_t units, blocks;     // blocks: an upper bound, by the block table
  int ctas;
  int64_t o_floats, ml_floats, prefix_ints, row_floats, score_floats;
  int64_t bytes() const {
    return 4 * (o_floats + ml_floats + row_floats + score_floats) + (4 * prefix_ints + 255) / 256 * 256;
  }
};

// false: a call that the kernel does not take
bool decode_plan(const CatcocKv4Call& c, bool weights, DecodePlan& d) {
  if (c.B <= 0 || c.B > 65536 || c.q_len <= 0 || c.q_len > 64 || c.Hk <= 0 || c.Hq <= 0 || c.Hq % c.Hk != 0 || (c.D != 64 && c.D != 128) || c.pages <= 0 ||
      c.max_pages <= 0 || c.window < 0 || c.sinks < 0 || static_cast<int64_t>(c.Hq / c.Hk) * c.q_len > 4096)
    return false;
  d.R = c.Hq / c.Hk * c.q_len;
  d.rows = d.R <= 4 && c.D == 128 ? 4 : d.R <= 8 ? 8 : 16;
  d.chunks = (d.R + d.rows - 1) / d.rows;
  d.units = static_cast<int64_t>(c.B) * c.Hk * d.chunks;
  int64_t seq = c.max_pages;
  if (c.window > 0) seq = std::min<int64_t>(seq, (static_cast<int64_t>(c.window) + c.q_len + 62) / 64 + 1 + (static_cast<int64_t>(c.sinks) + 63) / 64);
  d.blocks = d.units * seq;
  if (d.blocks > (1ll << 30) || static_cast<int64_t>(c.max_pages) * kPage > (1ll << 24)) return false;
  int device = 0;
  cudaGetDevice(&device);
  d.ctas = static_cast<int>(std::min<int64_t>(d.blocks, 2ll * catcoc_num_sms(device)));
  const int64_t pieces = d.ctas + d.units;
  d.o_floats = pieces * d.rows * c.D;
  d.ml_floats = pieces * d.rows * 2;
  d.prefix_ints = c.B + 1;
  d.row_floats = weights ? static_cast<int64_t>(c.B) * c.Hk * d.R * 2 : 0;
  d.score_floats = weights ? static_cast<int64_t>(c.B) * c.Hk * d.R * c.max_pages * kPage : 0;
  return true;
}
}  // namespace

extern "C" int64_t catcoc_kv4_decode_workspace_bytes(const CatcocKv4Call* c, int weights) {
  DecodePlan d;
  return c && decode_plan(*c, weights != 0, d) ? d.bytes() : -1;
}

extern "C" int catcoc_kv4_decode(const CatcocKv4Call* c, const void* q, const void* cache, const int* block_table, const int* kv_lens, void* out, float* weights,
                                 void* workspace, uint32_t* status, uint64_t timeout_ns, void* stream_) {
  DecodePlan d;
  if (!c || !q || !cache || !block_table || !kv_lens || !out || !workspace || !status || !decode_plan(*c, weights != nullptr, d)) {
    set_error("kv4_decode: bad arguments");
    return CATCOC_E_BAD_ARG;
  }
  const int B = c->B, Hk = c->Hk, D = c->D, fmt = c->fmt;
  if (fmt != CATCOC_FMT_F16 && fmt != CATCOC_FMT_BF16) { set_error("kv4_decode takes fp16 / bf16"); return CATCOC_E_UNSUPPORTED; }
  if (!(c->scale > 0.0f)) { set_error("kv4_decode: the softmax scale must be positive"); return CATCOC_E_UNSUPPORTED; }
  if (weights && c->S < c->max_pages * kPage) { set_error("kv4_decode: the weights are shorter than the block table's row"); return CATCOC_E_BAD_ARG; }
  if ((reinterpret_cast<uintptr_t>(q) | reinterpret_cast<uintptr_t>(cache) | reinterpret_cast<uintptr_t>(out) | reinterpret_cast<uintptr_t>(workspace)) & 15) {
    set_error("kv4_decode: buffers must be 16-byte aligned");
    return CATCOC_E_ALIGNMENT;
  }
  DecodeParams p;
  memset(&p, 0, sizeof(p));
  p.q = q; p.cache = static_cast<const uint8_t*>(cache); p.table = block_table; p.lens = kv_lens; p.out = out;
  p.part_o = static_cast<float*>(workspace);
  p.part_ml = p.part_o + d.o_floats;
  p.row_ml = p.part_ml + d.ml_floats;
  p.scores = p.row_ml + d.row_floats;
  p.prefix = reinterpret_cast<int*>(p.scores + d.score_floats);
  p.B = B; p.q_len = c->q_len; p.Hq = c->Hq; p.Hk = Hk; p.group = c->Hq / Hk; p.R = d.R; p.chunks = d.chunks;
  p.max_pages = c->max_pages; p.pages = c->pages; p.S = c->max_pages * kPage;
  p.window = std::min(c->window, 1 << 30); p.sinks = std::min(c->sinks, 1 << 30);   // (both beyond any length; their sums stay in range)
  p.scale_log2 = c->scale * 1.4426950408889634f;
  p.status = status;
  p.timeout_ns = timeout_ns ? timeout_ns : 10000000000ull;
  cudaStream_t stream = static_cast<cudaStream_t>(stream_);
  auto launch = [&](auto main_kernel, auto combine_kernel, size_t smem) -> int {
    CATCOC_CUDA_OK(cudaFuncSetAttribute(main_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(smem)));
    CATCOC_CUDA_OK(launch_overlapped(main_kernel, dim3(static_cast<unsigned>(d.ctas)), dim3(kThreads), smem, stream, p));
    CATCOC_CUDA_OK(launch_overlapped(combine_kernel, dim3(static_cast<unsigned>(d.units), static_cast<unsigned>((std::min(d.R, d.rows) + 3) / 4)), dim3(128), 0,
                                     stream, p, d.rows, d.ctas));
    if (weights) {
      const unsigned chunks = static_cast<unsigned>((p.S + 255) / 256), y = std::min(chunks, 32768u);
      CATCOC_CUDA_OK(launch_overlapped(kv4_weights_kernel, dim3(static_cast<unsigned>(B * Hk), y, (chunks + y - 1) / y), dim3(256), d.R * sizeof(float2), stream, p,
                                       weights, static_cast<int64_t>(c->S)));
    }
    return CATCOC_OK;
  };
  auto by_rows = [&](auto dim, auto type) -> int {
    constexpr int kD = decltype(dim)::value, kF = decltype(type)::value;
    auto with = [&](auto eights, auto pair) -> int {
      constexpr int kE = decltype(eights)::value;
      constexpr bool kP = decltype(pair)::value;
      return weights ? launch(kv4_decode_kernel<kD, kF, kE, kP, true>, kv4_combine_kernel<kD, kF, true>, sizeof(Smem<kD, kE, kP>))
                     : launch(kv4_decode_kernel<kD, kF, kE, kP, false>, kv4_combine_kernel<kD, kF, false>, sizeof(Smem<kD, kE, kP>));
    };
    if constexpr (kD == 128) {
      if (d.rows == 4) return with(std::integral_constant<int, 1>{}, std::true_type{});
    }
    return d.rows == 8 ? with(std::integral_constant<int, 1>{}, std::false_type{}) : with(std::integral_constant<int, 2>{}, std::false_type{});
  };
  const bool bf = fmt == CATCOC_FMT_BF16;
  if (D == 128) return bf ? by_rows(std::integral_constant<int, 128>{}, std::integral_constant<int, FMT_BF16>{}) : by_rows(std::integral_constant<int, 128>{}, std::integral_constant<int, FMT_F16>{});
  return bf ? by_rows(std::integral_constant<int, 64>{}, std::integral_constant<int, FMT_BF16>{}) : by_rows(std::integral_constant<int, 64>{}, std::integral_constant<int, FMT_F16>{});
}
