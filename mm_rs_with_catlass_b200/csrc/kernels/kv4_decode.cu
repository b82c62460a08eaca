// Attention of a decode step over the paged 4-bit cache (layout: catcoc/kv4.h).
//
// The query heads that share a KV head, and the new tokens of a sequence, are the rows of one unit; every code is read once for all
// of them. The blocks of all units form one list, by the lengths on the device, that is cut into equal runs over the CTAs; pieces
// of a unit that lies in several runs are merged by a second kernel, and a third one adds the probabilities to the caller's sums.
//
// The four warps of a CTA take half blocks (32 tokens) in turn, each with bulk copies, a softmax and an O of its own; they meet at the end of
// a unit. No warp waits for another one's copies, and none only copies.
//
// Both products run on codes, without their values: with scales and zeros constant over a group g of channels,
//   q . k_j = sum_g s_jg (sum_c q_c code_jc) + z_jg (sum_c q_c),   o_c = sum_j (p_j s_jg) code_jc + sum_j p_j z_jg,
// so that a code costs a mask (0.6 instructions, the values 4 tokens at a time 0.75): four bits at the bottom of a half are the
// subnormal code * 2^-24, those above them code * 2^-20, both exact operands. The 16 between them goes into q and into the result.
// q is brought into the range of a half by a power of two per row, p s by one per group that follows the largest scale, so
// that the only rounding in front of the accumulators is that of p s to 11 bits.
//
// S^T = K q^T has the tokens as rows; its accumulator, scaled, rounded and transposed by movmatrix, is the second operand of
// O^T += V^T (p s). Tokens fill the 16 rows of an instruction where query rows would fill a part of them.
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

constexpr int kWarps = 4;
constexpr int kThreads = 32 * kWarps;
constexpr int kTile = 16;                          // tokens of a matrix instruction
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
    if (s.sink < 0) s.sink = 0;
  }
  return s;
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

// Tokens of an item, what a warp takes at once: half a block, so that short runs keep the warps busy too
constexpr int kItem = 32;
constexpr int kSubs = kPage / kItem;

// A part of the run: blocks [i0, i1) of the n of a unit's list (Hk x chunks units a sequence)
struct Part {
  int b, unit, i0, i1, n;
};
// The next item of a warp and its part, which begins at `at` of the list
struct Ahead {
  Part part;
  int at, item, more;
};

template <int D, int NT>
struct Smem {
  using L = Block<D>;
  // an item: codes of K and of V, then their parameters
  static constexpr int kCodes = kItem * L::kRow, kPars = kItem * L::kParRow;
  static constexpr int kStageBytes = 2 * (kCodes + kPars);
  static constexpr int kStages = 2;    // of every warp
  alignas(128) uint8_t stage[kWarps][kStages][kStageBytes];
  float o[kWarps][8 * NT][D + 4];      // (4: the lanes of a warp store to different banks)
  float2 ml[kWarps][8 * NT];
  uint64_t full[kWarps][kStages];
  uint32_t abort_flag;
  uint32_t failed[kWarps];
  Ahead ahead[kWarps];
  int seqs[1];                         // [B + 1] blocks of the sequences before, then [B] lengths
};

// Row of a matrix instruction -> token of the tile. Two tokens of a pair are swapped in every other pair, so that the rows that four
// lanes read of V lie in both halves of the banks (K's stay free of conflicts).
CATCOC_DEVICE int token_of(int row) { return row ^ ((row >> 1) & 1); }

// D: head dimension, FMT: type of q and out, NT: query rows of a unit in eights, W: the scores are written for the weights
template <int D, int FMT, int NT, bool W>
__global__ void __launch_bounds__(kThreads, NT == 1 ? 4 : 3) kv4_decode_kernel(const __grid_constant__ DecodeParams p) {
  using L = Block<D>;
  using Sm = Smem<D, NT>;
  constexpr int G = L::kGroups, kRowsU = 8 * NT;
  extern __shared__ uint8_t smem_raw[];
  Sm& sm = *reinterpret_cast<Sm*>((reinterpret_cast<uintptr_t>(smem_raw) + 127) & ~static_cast<uintptr_t>(127));
  int* prefix = sm.seqs;
  int* seq_lens = sm.seqs + p.B + 1;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g8 = lane >> 2, t4 = lane & 3;
  volatile uint32_t* abort_flag = &sm.abort_flag;

  if (lane == 0) {
    for (int s = 0; s < Sm::kStages; ++s) ptx::mbar_init(&sm.full[warp][s], 1);
    if (warp == 0) sm.abort_flag = 0;
    ptx::mbar_fence_init();
  }
  ptx::grid_dependency_wait();
  ptx::launch_dependents();
  // blocks of the sequences before each one
  if (warp == 0) {
    int sum = 0;
    for (int base = 0; base < p.B; base += 32) {
      const int b = base + lane;
      int n = 0;
      if (b < p.B) {
        const int len = seq_len(p.lens, b, p.max_pages * kPage, p.status);
        seq_lens[b] = len;
        n = span_of(len, p.q_len, p.window, p.sinks).count();
      }
#pragma unroll
      for (int o = 1; o < 32; o *= 2) {
        const int y = __shfl_up_sync(0xffffffffu, n, o);
        if (lane >= o) n += y;
      }
      if (b < p.B) prefix[b + 1] = sum + n;
      sum += __shfl_sync(0xffffffffu, n, 31);
    }
    if (lane == 0) prefix[0] = 0;
    __syncwarp();
    if (blockIdx.x == 0)
      for (int b = lane; b <= p.B; b += 32) p.prefix[b] = prefix[b];
  }
  __syncthreads();
  const int per_seq = p.Hk * p.chunks;                            // units of a sequence
  const int total = prefix[p.B] * per_seq;
  const int per = (total + static_cast<int>(gridDim.x) - 1) / static_cast<int>(gridDim.x);
  const int begin = min(total, static_cast<int>(blockIdx.x) * per), end = min(total, begin + per);
  // the part of the run that begins at list position `at`, in sequence `b` or behind it
  auto part_at = [&](int at, int b) {
    while (prefix[b + 1] * per_seq <= at) ++b;
    const int n = prefix[b + 1] - prefix[b], in_seq = at - prefix[b] * per_seq, unit = in_seq / n, i0 = in_seq - unit * n;
    return Part{b, unit, i0, min(n, i0 + end - at), n};
  };
  int b0 = 0;                                                     // the last sequence that begins at or before `begin`
  for (int hi = p.B; hi - b0 > 1;) {
    const int mid = (b0 + hi) >> 1;
    if (prefix[mid] * per_seq <= begin) b0 = mid; else hi = mid;
  }

  // ------------------------------ copies ------------------------------
  // A warp fetches what it will work on, two items ahead and across parts. Item x of a part goes to warp x % 4. The name
  // of an item's block is read when the item before it is requested.
  // What it is at lies in shared memory: it is needed once an item, and the registers are short. (The name does not: a store
  // would wait for it.)
  Ahead& ahead = sm.ahead[warp];
  int requested = 0, ahead_page = -1;
  auto look = [&](Ahead a) {                                      // from a.at, a.item on to the next item of this warp
    while (!(a.more && a.item < (a.part.i1 - a.part.i0) * kSubs)) {
      if (a.more) a.at += a.part.i1 - a.part.i0;
      const int b = a.more ? a.part.b : b0;
      a.more = a.at < end;
      if (!a.more) break;
      a.part = part_at(a.at, b);
      a.item = warp;
    }
    if (a.more)
      ahead_page = p.table[static_cast<int64_t>(a.part.b) * p.max_pages + span_of(seq_lens[a.part.b], p.q_len, p.window, p.sinks).block(a.part.i0 + a.item / kSubs)];
    __syncwarp();
    if (lane == 0) ahead = a;
    __syncwarp();
  };
  auto request = [&] {
    Ahead a = ahead;
    if (!a.more) return;
    const int s = requested % Sm::kStages;
    uint64_t* bar = &sm.full[warp][s];
    if (lane == 0) {
      if (static_cast<uint32_t>(ahead_page) < static_cast<uint32_t>(p.pages)) {
        const uint8_t* src = p.cache + (static_cast<int64_t>(ahead_page) * p.Hk + a.part.unit / p.chunks) * L::kBytes;
        const int sub = a.item % kSubs;
        uint8_t* dst = sm.stage[warp][s];
        ptx::mbar_expect_tx(bar, Sm::kStageBytes);
#pragma unroll
        for (int half = 0; half < 2; ++half) {
          ptx::bulk_load_1d(dst + half * Sm::kCodes, src + half * L::kHalf + sub * Sm::kCodes, Sm::kCodes, bar);
          ptx::bulk_load_1d(dst + 2 * Sm::kCodes + half * Sm::kPars, src + half * L::kHalf + L::kPar + sub * Sm::kPars, Sm::kPars, bar);
        }
      } else {
        note(p.status, kErrPage, ahead_page, p.pages);                // what the stage held stands in for the block
        ptx::mbar_arrive(bar);
      }
    }
    ++requested;
    a.item += kWarps;
    look(a);
  };
  look(Ahead{{}, begin, 0, 0});
  for (int s = 0; s < Sm::kStages; ++s) request();

  // ------------------------------ products and softmax ------------------------------
  int taken = 0;
  bool ok = true;
  Part part{};
  for (int at = begin; at < end && ok; at += part.i1 - part.i0) {
    part = part_at(at, at > begin ? part.b : b0);
    const int b = part.b, len = seq_lens[b];
    const Span span = span_of(len, p.q_len, p.window, p.sinks);
    const int hk = part.unit / p.chunks, row0 = (part.unit - hk * p.chunks) * kRowsU;   // first row of the unit among the R of its head
    // q as the second operand of S^T: row g8 of every eight, the channels of this lane's words; b0, b1 of every step
    uint32_t qf[NT][2 * G][4];
    float qscale[NT][2], qsum[NT][G][2];              // of the rows of this lane's columns, 2 t4 and 2 t4 + 1: score = qscale * raw
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      const int r = row0 + nt * 8 + g8;
      const int tok = r / p.group;
      const uint16_t* src = static_cast<const uint16_t*>(p.q) + ((static_cast<int64_t>(b) * p.q_len + tok) * p.Hq + hk * p.group + (r - tok * p.group)) * D;
      float x[2 * G][8], mx = 0.0f, sum[G] = {};
#pragma unroll
      for (int i = 0; i < 2 * G; ++i) {
        uint4 raw = make_uint4(0, 0, 0, 0);
        if (r < p.R) raw = *reinterpret_cast<const uint4*>(src + (i % G) * 64 + (2 * t4 + i / G) * 8);
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
        qf[nt][i][0] = half2_of(x[i][0] * f, x[i][4] * f);
        qf[nt][i][1] = half2_of(x[i][1] * f * 0.0625f, x[i][5] * f * 0.0625f);
        qf[nt][i][2] = half2_of(x[i][2] * f, x[i][6] * f);
        qf[nt][i][3] = half2_of(x[i][3] * f * 0.0625f, x[i][7] * f * 0.0625f);
      }
      const float back = p.scale_log2 * 16777216.0f / f;
#pragma unroll
      for (int g = 0; g < G; ++g) {
        sum[g] += __shfl_xor_sync(0xffffffffu, sum[g], 1);
        sum[g] += __shfl_xor_sync(0xffffffffu, sum[g], 2);
        sum[g] *= f * (1.0f / 16777216.0f);           // in the unit of the products of codes
      }
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        const int from = (2 * t4 + c) * 4;
        qscale[nt][c] = __shfl_sync(0xffffffffu, back, from);
#pragma unroll
        for (int g = 0; g < G; ++g) qsum[nt][g][c] = __shfl_sync(0xffffffffu, sum[g], from);
      }
    }
    // m: largest raw score, as far as it is followed; m_neg: minus its score; limit: raw score from which on it moves
    float o[NT][G][4][4] = {}, m[NT][2], m_neg[NT][2], limit[NT][2], l[NT][2] = {}, zsum[NT][G][2] = {};
    int e_ref[G];                                     // exponent field that the scales of V are held against
    float vscale[G];                                  // 2^(kPShift + 127 - e_ref)
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int c = 0; c < 2; ++c) { m[nt][c] = limit[nt][c] = -INFINITY; m_neg[nt][c] = 0.0f; }
#pragma unroll
    for (int g = 0; g < G; ++g) { e_ref[g] = 8; vscale[g] = __uint_as_float((254u + kPShift - 8u) << 23); }
    const int pos_lo = len - p.q_len, pos_hi = len - 1;

    // TILES tiles from token `t0` of the stage on. ALL: every row sees every key of them.
    auto tiles = [&](auto all_c, auto count_c, const uint8_t* st, int t0, int key0) {
      constexpr bool ALL = decltype(all_c)::value;
      constexpr int TILES = decltype(count_c)::value;
      const uint8_t *kc = st + t0 * L::kRow, *vc = kc + Sm::kCodes, *kp = st + 2 * Sm::kCodes + t0 * L::kParRow, *vp = kp + Sm::kPars;
      float s[TILES][NT][4];
      uint32_t vpar[TILES][2][G];
      const int tk = token_of(g8);
#pragma unroll
      for (int i = 0; i < TILES; ++i) {
        // S^T: rows g8 and g8 + 8 are tokens, channels by t4; one accumulator per group
        uint32_t ka[2 * G], kb[2 * G], par[2][G];
        const uint8_t* at = kc + (i * kTile + tk) * L::kRow + t4 * 8 * G;
        if constexpr (G == 2) {
          const uint4 a = *reinterpret_cast<const uint4*>(at), c = *reinterpret_cast<const uint4*>(at + 8 * L::kRow);
          ka[0] = a.x; ka[1] = a.y; ka[2] = a.z; ka[3] = a.w;
          kb[0] = c.x; kb[1] = c.y; kb[2] = c.z; kb[3] = c.w;
        } else {
          const uint2 a = *reinterpret_cast<const uint2*>(at), c = *reinterpret_cast<const uint2*>(at + 8 * L::kRow);
          ka[0] = a.x; ka[1] = a.y;
          kb[0] = c.x; kb[1] = c.y;
        }
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          const int off = (i * kTile + tk + 8 * u) * L::kParRow;
          if constexpr (G == 2) {
            const uint2 a = *reinterpret_cast<const uint2*>(kp + off), c = *reinterpret_cast<const uint2*>(vp + off);
            par[u][0] = a.x; par[u][1] = a.y; vpar[i][u][0] = c.x; vpar[i][u][1] = c.y;
          } else {
            par[u][0] = *reinterpret_cast<const uint32_t*>(kp + off); vpar[i][u][0] = *reinterpret_cast<const uint32_t*>(vp + off);
          }
        }
        float acc[NT][G][4] = {};
#pragma unroll
        for (int w = 0; w < 2 * G; ++w) {
          const uint32_t a8 = ka[w] >> 8, b8 = kb[w] >> 8;
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) {
            mma_f16(acc[nt][w % G], ka[w] & 0x000f000fu, kb[w] & 0x000f000fu, ka[w] & 0x00f000f0u, kb[w] & 0x00f000f0u, qf[nt][w][0], qf[nt][w][1]);
            mma_f16(acc[nt][w % G], a8 & 0x000f000fu, b8 & 0x000f000fu, a8 & 0x00f000f0u, b8 & 0x00f000f0u, qf[nt][w][2], qf[nt][w][3]);
          }
        }
        // raw scores of tokens g8 ([0], [1]) and g8 + 8 ([2], [3]), columns 2 t4 and 2 t4 + 1
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const int u = e >> 1, c = e & 1;
            float a = bf16_hi(par[u][0]) * qsum[nt][0][c];
#pragma unroll
            for (int g = 1; g < G; ++g) a = fmaf(bf16_hi(par[u][g]), qsum[nt][g][c], a);
#pragma unroll
            for (int g = 0; g < G; ++g) a = fmaf(bf16_lo(par[u][g]), acc[nt][g][e], a);
            s[i][nt][e] = a;
          }
        if constexpr (!ALL) {
          // what a row does not see weighs nothing, whatever the cache holds there
          bool seen[2] = {false, false};
#pragma unroll
          for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const int r = row0 + nt * 8 + 2 * t4 + (e & 1);
              const bool v = r < p.R && sees(pos_lo + r / p.group, key0 + i * kTile + tk + 8 * (e >> 1), p.window, p.sinks);
              if (!v) s[i][nt][e] = -INFINITY;
              seen[e >> 1] |= v;
            }
#pragma unroll
          for (int u = 0; u < 2; ++u)
#pragma unroll
            for (int g = 0; g < G; ++g)
              if (!seen[u]) vpar[i][u][g] = 0u;
        }
        if constexpr (W) {
          float* dst = p.scores + (static_cast<int64_t>(b) * p.Hk + hk) * p.R * p.S + key0 + i * kTile + tk;
#pragma unroll
          for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int c = 0; c < 2; ++c) {
              const int r = row0 + nt * 8 + 2 * t4 + c;
              if (r < p.R) {
                dst[static_cast<int64_t>(r) * p.S] = s[i][nt][c] * qscale[nt][c];
                dst[static_cast<int64_t>(r) * p.S + 8] = s[i][nt][2 + c] * qscale[nt][c];
              }
            }
        }
      }
      // the references: m moves when a score exceeds its own by more than 8, e_ref when a scale is past twice its power
      float ps[TILES][G][2], top = 0.0f;
      bool move = false;
#pragma unroll
      for (int i = 0; i < TILES; ++i)
#pragma unroll
        for (int g = 0; g < G; ++g)
#pragma unroll
          for (int u = 0; u < 2; ++u) {
            ps[i][g][u] = bf16_lo(vpar[i][u][g]) * vscale[g];
            top = fmaxf(top, ps[i][g][u]);
          }
      move = top >= static_cast<float>(2 << kPShift);
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
        float beta[G];
#pragma unroll
        for (int g = 0; g < G; ++g) {
          // (scales are not negative; one that is no number, or infinite, sets no reference)
          uint32_t ex = 0;
#pragma unroll
          for (int i = 0; i < TILES; ++i)
#pragma unroll
            for (int u = 0; u < 2; ++u) {
              const uint32_t x = (vpar[i][u][g] >> 7) & 0xffu;
              ex = max(ex, x == 255u ? 0u : x);
            }
          const int e_new = max(e_ref[g], static_cast<int>(__reduce_max_sync(0xffffffffu, ex)));
          beta[g] = e_new - e_ref[g] > 126 ? 0.0f : __uint_as_float(static_cast<uint32_t>(127 + e_ref[g] - e_new) << 23);
          e_ref[g] = e_new;
          vscale[g] = __uint_as_float((254u + kPShift - static_cast<uint32_t>(e_new)) << 23);
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
            for (int g = 0; g < G; ++g) {
              zsum[nt][g][c] *= alpha;
#pragma unroll
              for (int k = 0; k < 4; ++k) {
                o[nt][g][k][c] *= alpha * beta[g];
                o[nt][g][k][2 + c] *= alpha * beta[g];
              }
            }
          }
      }
#pragma unroll
      for (int i = 0; i < TILES; ++i) {
        uint32_t pb[NT][G][2];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
          float pr[4];
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            pr[e] = ptx::ex2_approx(fmaf(s[i][nt][e], qscale[nt][e & 1], m_neg[nt][e & 1]));
            l[nt][e & 1] += pr[e];
          }
#pragma unroll
          for (int g = 0; g < G; ++g) {
            float w[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              w[e] = pr[e] * ps[i][g][e >> 1];
              float z = bf16_hi(vpar[i][e >> 1][g]);
              if (!ALL && s[i][nt][e] == -INFINITY) { w[e] = 0.0f; z = 0.0f; }
              zsum[nt][g][e & 1] = fmaf(pr[e], z, zsum[nt][g][e & 1]);
            }
            pb[nt][g][0] = transpose8(half2_of(w[0], w[1]));
            pb[nt][g][1] = transpose8(half2_of(w[2], w[3]));
          }
        }
        // O^T: rows g8 and g8 + 8 are the channels 64 g + 8 g8 + 2 k and + 1, tokens of the rows 2 t4, 2 t4 + 1, + 8, + 9
        uint32_t vw[4][G];
#pragma unroll
        for (int u = 0; u < 4; ++u) {
          const uint8_t* at = vc + (i * kTile + token_of(2 * t4 + (u & 1)) + 8 * (u >> 1)) * L::kRow + g8 * 4 * G;
          if constexpr (G == 2) { const uint2 x = *reinterpret_cast<const uint2*>(at); vw[u][0] = x.x; vw[u][1] = x.y; }
          else vw[u][0] = *reinterpret_cast<const uint32_t*>(at);
        }
#pragma unroll
        for (int g = 0; g < G; ++g)
#pragma unroll
          for (int hw = 0; hw < 2; ++hw) {
            const uint32_t x = __byte_perm(vw[0][g], vw[1][g], hw ? 0x7632 : 0x5410), y = __byte_perm(vw[2][g], vw[3][g], hw ? 0x7632 : 0x5410);
            const uint32_t x8 = x >> 8, y8 = y >> 8;
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
              mma_f16(o[nt][g][2 * hw], x & 0x000f000fu, x & 0x00f000f0u, y & 0x000f000fu, y & 0x00f000f0u, pb[nt][g][0], pb[nt][g][1]);
              mma_f16(o[nt][g][2 * hw + 1], x8 & 0x000f000fu, x8 & 0x00f000f0u, y8 & 0x000f000fu, y8 & 0x00f000f0u, pb[nt][g][0], pb[nt][g][1]);
            }
          }
      }
    };

    for (int item = warp; item < (part.i1 - part.i0) * kSubs; item += kWarps) {
      const int st = taken % Sm::kStages;
      ok = ptx::mbar_wait(&sm.full[warp][st], static_cast<uint32_t>(taken / Sm::kStages) & 1u, p.timeout_ns, abort_flag);
      if (!ok) break;
      ++taken;
      const int key0 = span.block(part.i0 + item / kSubs) * kPage + (item % kSubs) * kItem;
      const uint8_t* stage = sm.stage[warp][st];
      if (key0 + kItem - 1 <= pos_lo && (p.window == 0 || pos_hi - key0 < p.window || key0 + kItem <= p.sinks)) {
        if constexpr (NT == 1) {
          tiles(std::true_type{}, std::integral_constant<int, 2>{}, stage, 0, key0);
        } else {
#pragma unroll 1
          for (int t = 0; t < kItem; t += kTile) tiles(std::true_type{}, std::integral_constant<int, 1>{}, stage, t, key0 + t);
        }
      } else {
#pragma unroll 1
        for (int t = 0; t < kItem; t += kTile) {
          const int k0 = key0 + t;
          if (k0 <= pos_hi && (p.window == 0 || pos_lo - (k0 + kTile - 1) < p.window || k0 < p.sinks))
            tiles(std::false_type{}, std::integral_constant<int, 1>{}, stage, t, k0);
        }
      }
      __syncwarp();
      request();                                       // into the stage that was just read
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
          for (int g = 0; g < G; ++g) zsum[nt][g][c] += __shfl_xor_sync(0xffffffffu, zsum[nt][g][c], d);
        }
        // (from here on m is a score)
        m[nt][c] = m[nt][c] == -INFINITY ? -INFINITY : -m_neg[nt][c];
        if (g8 == 0) sm.ml[warp][nt * 8 + 2 * t4 + c] = make_float2(m[nt][c], l[nt][c]);
      }
    if (!ok && lane == 0) *abort_flag = 1;
    if (lane == 0) sm.failed[warp] = ok ? 0u : 1u;
    // (every warp walks the same parts and takes all barriers, also after a failed wait; all leave together)
    __syncthreads();
    ok = (sm.failed[0] | sm.failed[1] | sm.failed[2] | sm.failed[3]) == 0u;
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        const int r = nt * 8 + 2 * t4 + c;
        float mt = sm.ml[0][r].x;
#pragma unroll
        for (int w = 1; w < kWarps; ++w) mt = fmaxf(mt, sm.ml[w][r].x);
        const float a = m[nt][c] == -INFINITY ? 0.0f : ptx::ex2_approx(m[nt][c] - mt);
#pragma unroll
        for (int g = 0; g < G; ++g) {
          // 2^24 and 2^(e_ref - 127 - 5) undone in two steps: either alone could leave the range
          const float f1 = __uint_as_float(static_cast<uint32_t>(e_ref[g]) << 23), f2 = a * (16777216.0f / (1 << kPShift));
          float4 v[2];
          float* f = reinterpret_cast<float*>(v);
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            f[2 * k] = fmaf(o[nt][g][k][c] * f2, f1, a * zsum[nt][g][c]);
            f[2 * k + 1] = fmaf(o[nt][g][k][2 + c] * (f2 * 0.0625f), f1, a * zsum[nt][g][c]);
          }
          // (a warp that saw nothing of a row has nothing to add, not zero times what it holds)
          if (m[nt][c] == -INFINITY && l[nt][c] == 0.0f) v[0] = v[1] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
          float4* dst = reinterpret_cast<float4*>(&sm.o[warp][r][g * 64 + g8 * 8]);
          dst[0] = v[0];
          dst[1] = v[1];
        }
      }
    __syncthreads();
    if (!ok) break;
    // thread: eight columns of a row
    const bool alone = part.i1 - part.i0 == part.n;
    for (int x = threadIdx.x; x < kRowsU * (D / 8); x += kThreads) {
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
        const float4 a = *reinterpret_cast<const float4*>(&sm.o[w][r][col]), c = *reinterpret_cast<const float4*>(&sm.o[w][r][col + 4]);
        v[0] += a.x; v[1] += a.y; v[2] += a.z; v[3] += a.w;
        v[4] += c.x; v[5] += c.y; v[6] += c.z; v[7] += c.w;
      }
      if (alone) {
        const float inv = lt == 0.0f ? 0.0f : 1.0f / lt;
        const int tok = rr / p.group;
        uint16_t* dst = static_cast<uint16_t*>(p.out) + ((static_cast<int64_t>(b) * p.q_len + tok) * p.Hq + hk * p.group + (rr - tok * p.group)) * D + col;
        ptx::st_global_v4(dst, make_uint4(attn::pack16<FMT>(v[0] * inv, v[1] * inv), attn::pack16<FMT>(v[2] * inv, v[3] * inv),
                                          attn::pack16<FMT>(v[4] * inv, v[5] * inv), attn::pack16<FMT>(v[6] * inv, v[7] * inv)));
        if (W && col == 0) *reinterpret_cast<float2*>(p.row_ml + ((static_cast<int64_t>(b) * p.Hk + hk) * p.R + rr) * 2) = make_float2(mt, lt);
      } else {
        const int64_t piece = (static_cast<int64_t>(blockIdx.x) + b * per_seq + part.unit) * kRowsU + r;
        float4* dst = reinterpret_cast<float4*>(p.part_o + piece * D + col);
        dst[0] = make_float4(v[0], v[1], v[2], v[3]);
        dst[1] = make_float4(v[4], v[5], v[6], v[7]);
        if (col == 0) *reinterpret_cast<float2*>(p.part_ml + piece * 2) = make_float2(mt, lt);
      }
    }
    __syncthreads();                                   // the next part's pieces overwrite these
  }
  if (!ok) {
    // the run was given up: this warp's copies land before the block's memory is handed on; noted once for the launch
    volatile uint32_t never = 0;
    for (int i = taken; i < requested; ++i)
      ptx::mbar_wait(&sm.full[warp][i % Sm::kStages], static_cast<uint32_t>(i / Sm::kStages) & 1u, 100000000ull, &never);
    if (threadIdx.x == 0 && atomicCAS(p.status, 0u, static_cast<uint32_t>(STATUS_TIMEOUT_PIPELINE)) == 0u) {
      p.status[1] = 0u; p.status[2] = 400u; p.status[3] = 0u; p.status[4] = 0u; p.status[5] = 0u; p.status[6] = blockIdx.x;
      __threadfence_system();
    }
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
  const int n = p.prefix[b + 1] - p.prefix[b], total = p.prefix[p.B] * per_seq, per = (total + ctas - 1) / ctas;
  const int first = p.prefix[b] * per_seq + in_seq * n;
  const int tok = rr / p.group;
  uint16_t* dst = static_cast<uint16_t*>(p.out) + ((static_cast<int64_t>(b) * p.q_len + tok) * p.Hq + hk * p.group + (rr - tok * p.group)) * D + lane * kPer;
  float m = -INFINITY, l = 0.0f, acc[kPer] = {};
  if (n > 0) {
    const int c0 = first / per, c1 = (first + n - 1) / per;
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
  const int j = blockIdx.y * 256 + threadIdx.x;
  if (static_cast<int>(blockIdx.y) * 256 >= len) return;
  for (int r = threadIdx.x; r < p.R; r += 256) {
    const float2 ml = *reinterpret_cast<const float2*>(p.row_ml + (static_cast<int64_t>(bh) * p.R + r) * 2);
    row[r] = make_float2(ml.x == -INFINITY ? 0.0f : ml.x, ml.y == 0.0f ? 0.0f : 1.0f / ml.y);
  }
  __syncthreads();
  if (j >= len) return;
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
  int R, nt, chunks;
  int64_t units, blocks;     // blocks: an upper bound, by the block table
  int ctas;
  int64_t o_floats, ml_floats, prefix_ints, row_floats, score_floats;
  int64_t bytes() const {
    return 4 * (o_floats + ml_floats + row_floats + score_floats) + (4 * prefix_ints + 255) / 256 * 256;
  }
};

// false: a call that the kernel does not take
bool decode_plan(const CatcocKv4Call& c, bool weights, DecodePlan& d) {
  if (c.B <= 0 || c.B > 4096 || c.q_len <= 0 || c.q_len > 64 || c.Hk <= 0 || c.Hq <= 0 || c.Hq % c.Hk != 0 || (c.D != 64 && c.D != 128) || c.pages <= 0 ||
      c.max_pages <= 0 || c.window < 0 || c.sinks < 0 || static_cast<int64_t>(c.Hq / c.Hk) * c.q_len > 4096)
    return false;
  d.R = c.Hq / c.Hk * c.q_len;
  d.nt = d.R <= 8 ? 1 : 2;
  d.chunks = (d.R + 8 * d.nt - 1) / (8 * d.nt);
  d.units = static_cast<int64_t>(c.B) * c.Hk * d.chunks;
  int64_t seq = c.max_pages;
  if (c.window > 0) seq = std::min<int64_t>(seq, (static_cast<int64_t>(c.window) + c.q_len + 62) / 64 + 1 + (static_cast<int64_t>(c.sinks) + 63) / 64);
  d.blocks = d.units * seq;
  if (d.blocks > (1ll << 30) || static_cast<int64_t>(c.max_pages) * kPage > (1ll << 24)) return false;
  int device = 0;
  cudaGetDevice(&device);
  d.ctas = static_cast<int>(std::min<int64_t>(d.blocks, static_cast<int64_t>(catcoc_num_sms(device)) * (d.nt == 1 ? 4 : 3)));
  const int64_t pieces = d.ctas + d.units, rows = 8 * d.nt;
  d.o_floats = pieces * rows * c.D;
  d.ml_floats = pieces * rows * 2;
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
    smem += static_cast<size_t>(B) * 8 + 128;
    CATCOC_CUDA_OK(cudaFuncSetAttribute(main_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(smem)));
    CATCOC_CUDA_OK(launch_overlapped(main_kernel, dim3(static_cast<unsigned>(d.ctas)), dim3(kThreads), smem, stream, p));
    CATCOC_CUDA_OK(launch_overlapped(combine_kernel, dim3(static_cast<unsigned>(d.units), static_cast<unsigned>((std::min(d.R, 8 * d.nt) + 3) / 4)), dim3(128), 0,
                                     stream, p, 8 * d.nt, d.ctas));
    if (weights)
      CATCOC_CUDA_OK(launch_overlapped(kv4_weights_kernel, dim3(static_cast<unsigned>(B * Hk), static_cast<unsigned>((p.S + 255) / 256)), dim3(256),
                                       d.R * sizeof(float2), stream, p, weights, static_cast<int64_t>(c->S)));
    return CATCOC_OK;
  };
  auto by_rows = [&](auto dim, auto type) -> int {
    constexpr int kD = decltype(dim)::value, kF = decltype(type)::value;
    if (d.nt == 1)
      return weights ? launch(kv4_decode_kernel<kD, kF, 1, true>, kv4_combine_kernel<kD, kF, true>, sizeof(Smem<kD, 1>))
                     : launch(kv4_decode_kernel<kD, kF, 1, false>, kv4_combine_kernel<kD, kF, false>, sizeof(Smem<kD, 1>));
    return weights ? launch(kv4_decode_kernel<kD, kF, 2, true>, kv4_combine_kernel<kD, kF, true>, sizeof(Smem<kD, 2>))
                   : launch(kv4_decode_kernel<kD, kF, 2, false>, kv4_combine_kernel<kD, kF, false>, sizeof(Smem<kD, 2>));
  };
  const bool bf = fmt == CATCOC_FMT_BF16;
  if (D == 128) return bf ? by_rows(std::integral_constant<int, 128>{}, std::integral_constant<int, FMT_BF16>{}) : by_rows(std::integral_constant<int, 128>{}, std::integral_constant<int, FMT_F16>{});
  return bf ? by_rows(std::integral_constant<int, 64>{}, std::integral_constant<int, FMT_BF16>{}) : by_rows(std::integral_constant<int, 64>{}, std::integral_constant<int, FMT_F16>{});
}
