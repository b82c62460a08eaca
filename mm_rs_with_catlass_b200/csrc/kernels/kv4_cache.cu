// The 4-bit key / value cache on its way in, out and through an eviction (layout and formulas: catcoc/kv4.h). All of it is bound
// by bytes: 16-bit values in and 4.5 bits out or the reverse, and 4.5 bits of every kept token moved.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <algorithm>

#include "catcoc/capi.h"
#include "catcoc/host_util.h"
#include "catcoc/kv4.h"
#include "catcoc/params.h"
#include "catcoc/ptx.cuh"

using namespace catcoc;
using namespace catcoc::host;
using namespace catcoc::kv4;

namespace {

template <int FMT>
CATCOC_DEVICE uint32_t pack2(float lo, float hi) {
  if constexpr (FMT == FMT_BF16) { __nv_bfloat162 h = __floats2bfloat162_rn(lo, hi); return *reinterpret_cast<uint32_t*>(&h); }
  else { __half2 h = __floats2half2_rn(lo, hi); return *reinterpret_cast<uint32_t*>(&h); }
}

// ------------------------------------------------------------- append -------------------------------------------------------------

struct AppendParams {
  const void *k, *v;             // [T, Hk, D], a token's pitch and a head's pitch in elements
  int64_t k_token, k_head, v_token, v_head;
  uint8_t* cache;
  const int *table, *lens, *ends;
  int T, B, Hk, q_len, max_pages, pages;
  uint32_t* status;
};

template <int FMT>
CATCOC_DEVICE uint32_t min2_nan(uint32_t a, uint32_t b) {
  uint32_t r;
  if constexpr (FMT == FMT_BF16) asm("min.NaN.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  else asm("min.NaN.f16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  return r;
}
template <int FMT>
CATCOC_DEVICE uint32_t max2_nan(uint32_t a, uint32_t b) {
  uint32_t r;
  if constexpr (FMT == FMT_BF16) asm("max.NaN.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  else asm("max.NaN.f16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  return r;
}

// Words of sixteen channels and the parameters of their group, whose other 48 channels are in the lanes `lane ^ 1` and `lane ^ 2`.
// The extremes are taken in pairs of the input's own type, as (min, -max) they travel in one register.
template <int FMT>
CATCOC_DEVICE void quantise(const uint4 (&raw)[2], uint32_t (&word)[2], uint32_t& param) {
  const uint32_t u[8] = {raw[0].x, raw[0].y, raw[0].z, raw[0].w, raw[1].x, raw[1].y, raw[1].z, raw[1].w};
  uint32_t lo2 = u[0], hi2 = u[0];
#pragma unroll
  for (int i = 1; i < 8; ++i) {
    lo2 = min2_nan<FMT>(lo2, u[i]);
    hi2 = max2_nan<FMT>(hi2, u[i]);
  }
  // (min of the even ones, -max of the even ones) and the same of the odd ones
  uint32_t m = min2_nan<FMT>(__byte_perm(lo2, hi2, 0x5410) ^ 0x80000000u, __byte_perm(lo2, hi2, 0x7632) ^ 0x80000000u);
  m = min2_nan<FMT>(m, __shfl_xor_sync(0xffffffffu, m, 1));
  m = min2_nan<FMT>(m, __shfl_xor_sync(0xffffffffu, m, 2));
  float lo, hi;
  if constexpr (FMT == FMT_BF16) {
    lo = bf16_lo(m);
    hi = -bf16_hi(m);
  } else {
    const float2 v = __half22float2(*reinterpret_cast<const __half2*>(&m));
    lo = v.x;
    hi = -v.y;
  }
  // each rounding is the cache's own: the scale and the zero are held in bf16, and the codes are taken against the rounded ones
  float s = __bfloat162float(__float2bfloat16_rn((hi - lo) * (1.0f / 15.0f)));
  const float z = __bfloat162float(__float2bfloat16_rn(lo));
  if (s < 1.17549435e-38f) s = 0.0f;                   // a group of one value, or a range whose reciprocal would overflow
  if (!(s <= 3.4e38f)) s = __uint_as_float(0x7fc00000u);   // a NaN, an infinity, or a range past all numbers
  const float r = s > 0.0f ? 1.0f / s : 0.0f;
  param = (__float_as_uint(s) >> 16) | (__float_as_uint(z) & 0xffff0000u);
  // rint by the rounding of a sum with 1.5 * 2^23, whose last bits are then the code; the words are sums of these numbers times 16^n,
  // less what the sums hold of 1.5 * 2^23 itself
  constexpr uint32_t kBias = 0x4b400000u;
  constexpr float kMagic = 12582912.0f;
  const uint64_t z2 = ptx::pack_f32x2(-z, -z), r2 = ptx::pack_f32x2(r, r), magic2 = ptx::pack_f32x2(kMagic, kMagic), none = ptx::pack_f32x2(-0.0f, -0.0f);
#pragma unroll
  for (int w = 0; w < 2; ++w) {
    uint32_t sum = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      float x0, x1;
      if constexpr (FMT == FMT_BF16) {
        x0 = bf16_lo(u[4 * w + i]);
        x1 = bf16_hi(u[4 * w + i]);
      } else {
        const float2 v = __half22float2(*reinterpret_cast<const __half2*>(&u[4 * w + i]));
        x0 = v.x;
        x1 = v.y;
      }
      ptx::unpack_f32x2(ptx::fma_f32x2(ptx::add_f32x2(ptx::pack_f32x2(x0, x1), z2), r2, none), x0, x1);
      // a NaN becomes 0. (bf16: the zero is the least value itself, and 15 scales fall short of the range by less than half of one.)
      x0 = fmaxf(x0, 0.0f);
      x1 = fmaxf(x1, 0.0f);
      if constexpr (FMT == FMT_F16) {
        x0 = fminf(x0, 15.0f);
        x1 = fminf(x1, 15.0f);
      }
      ptx::unpack_f32x2(ptx::add_f32x2(ptx::pack_f32x2(x0, x1), magic2), x0, x1);
      sum += (__float_as_uint(x0) << (8 * i)) + (__float_as_uint(x1) << (8 * i + 4));
    }
    constexpr uint32_t kHeld = kBias * 0x11111111u;     // sum of kBias * 16^n, n = 0..7
    word[w] = sum - kHeld;
  }
}

// A thread: sixteen channels of K and of V of one token and head; 4 G lanes make a row.
template <int D, int FMT>
__global__ void __launch_bounds__(256) kv4_append_kernel(const AppendParams p) {
  using L = Block<D>;
  constexpr int G = L::kGroups, kLanes = 4 * G;
  ptx::grid_dependency_wait();
  const int lane = threadIdx.x & 31;
  const int64_t idx = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x;
  const int64_t rows = static_cast<int64_t>(p.T) * p.Hk;
  const int64_t row = idx / kLanes;
  const int j = static_cast<int>(idx % kLanes), g = j / 4, w = 2 * (j % 4);     // channels 64 g + 8 w + (0..15)
  const bool real = row < rows;
  const int t = real ? static_cast<int>(row / p.Hk) : p.T, h = real ? static_cast<int>(row - static_cast<int64_t>(t) * p.Hk) : 0;
  uint4 kr[2] = {}, vr[2] = {};
  if (real) {
    const int c = g * 64 + w * 8;
    const uint4* ks = reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(p.k) + t * p.k_token + h * p.k_head + c);
    const uint4* vs = reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(p.v) + t * p.v_token + h * p.v_head + c);
    kr[0] = ks[0]; kr[1] = ks[1];
    vr[0] = vs[0]; vr[1] = vs[1];
  }
  // the token's sequence: how many of the sequences end at or before it
  int b, behind;                                         // `behind`: tokens of the sequence from this one on
  if (p.ends == nullptr) {
    b = t / p.q_len;
    behind = (b + 1) * p.q_len - t;
  } else {
    b = 0;
    behind = 0;
    for (int base = 0; base < p.B; base += 32) {
      const int e = base + lane < p.B ? p.ends[base + lane] : 0x7fffffff;
      int n = 0;                                         // entries of this chunk that are <= t: ends ascend
#pragma unroll
      for (int step = 16; step > 0; step >>= 1) {
        const int at = __shfl_sync(0xffffffffu, e, n + step - 1);
        if (at <= t) n += step;
      }
      const int last = __shfl_sync(0xffffffffu, e, n);
      if (n == 31 && last <= t) n = 32;
      const int mine = __shfl_sync(0xffffffffu, e, n & 31);
      if (behind == 0) {
        b = base + n;
        if (n < 32) behind = mine == 0x7fffffff ? -1 : mine - t;
      }
    }
  }
  uint32_t kp, vp, kw[2], vw[2];
  quantise<FMT>(kr, kw, kp);
  quantise<FMT>(vr, vw, vp);
  if constexpr (G == 2) {
    // words w and w + 1 of a group are two words apart in the row: the lanes of the two groups exchange one, and each has two in a row
    auto exchange = [&](uint32_t (&x)[2]) {
      const uint32_t got = __shfl_xor_sync(0xffffffffu, g == 0 ? x[1] : x[0], 4);
      if (g == 0) x[1] = got;
      else x[0] = got;
    };
    exchange(kw);
    exchange(vw);
  }
  if (!real || b >= p.B || behind <= 0) return;           // a token behind the last sequence
  // (from the length as it is: counted from one that is cut to the table's row, the token would land on one of the sequence's last)
  const int len = p.lens[b];
  const int64_t at_pos = static_cast<int64_t>(len) - behind;
  if (at_pos < 0 || at_pos >= p.max_pages * kPage) { if (j == 0) note(p.status, kErrLen, len, at_pos < 0 ? behind : p.max_pages * kPage); return; }
  const int pos = static_cast<int>(at_pos);
  const int page = page_of(p.table, static_cast<int64_t>(b) * p.max_pages, pos / kPage, p.pages, p.status);
  if (page < 0) return;
  uint8_t* block = p.cache + (static_cast<int64_t>(page) * p.Hk + h) * L::kBytes;
  const int slot = pos % kPage, at = G == 2 ? 2 * w + 2 * g : w;   // first of this lane's two words
  *reinterpret_cast<uint2*>(block + slot * L::kRow + at * 4) = make_uint2(kw[0], kw[1]);
  *reinterpret_cast<uint2*>(block + L::kHalf + slot * L::kRow + at * 4) = make_uint2(vw[0], vw[1]);
  if (w == 0) *reinterpret_cast<uint32_t*>(block + L::kPar + slot * L::kParRow + g * 4) = kp;
  if (w == 2) *reinterpret_cast<uint32_t*>(block + L::kHalf + L::kPar + slot * L::kParRow + g * 4) = vp;
}

// ------------------------------------------------------------- read -------------------------------------------------------------

struct ReadParams {
  const uint8_t* cache;
  const int *table, *lens, *start;
  void *k, *v;                   // [B, Hk, count, D]
  int B, Hk, count, max_pages, pages;
  uint32_t* status;
};

template <int FMT>
CATCOC_DEVICE uint4 values(uint32_t word, uint32_t param) {
  const float s = bf16_lo(param), z = bf16_hi(param);
  // a code in the last bits of 2^23 is a whole number of a float without a conversion
  auto code = [&](int i) { return __uint_as_float(0x4b000000u | ((word >> (4 * i)) & 15u)) - 8388608.0f; };
  uint32_t o[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) o[i] = pack2<FMT>(fmaf(s, code(2 * i), z), fmaf(s, code(2 * i + 1), z));
  return make_uint4(o[0], o[1], o[2], o[3]);
}

// A thread: word w of every group of one token, K and V.
template <int D, int FMT>
__global__ void __launch_bounds__(256) kv4_read_kernel(const ReadParams p) {
  using L = Block<D>;
  constexpr int G = L::kGroups;
  ptx::grid_dependency_wait();
  const int w = threadIdx.x & 7;
  const int64_t i = static_cast<int64_t>(blockIdx.y) * 32 + (threadIdx.x >> 3);
  if (i >= p.count) return;
  const int b = blockIdx.x / p.Hk, h = blockIdx.x - b * p.Hk;
  const int len = seq_len(p.lens, b, p.max_pages * kPage, p.status);
  const int64_t pos = (p.start != nullptr ? p.start[b] : 0) + i;
  uint32_t kw[G] = {}, vw[G] = {}, kp[G] = {}, vp[G] = {};
  if (pos >= 0 && pos < len) {
    const int page = page_of(p.table, static_cast<int64_t>(b) * p.max_pages, static_cast<int>(pos / kPage), p.pages, p.status);
    if (page >= 0) {
      const uint8_t* block = p.cache + (static_cast<int64_t>(page) * p.Hk + h) * L::kBytes;
      const int slot = static_cast<int>(pos % kPage);
#pragma unroll
      for (int g = 0; g < G; ++g) {
        kw[g] = reinterpret_cast<const uint32_t*>(block + slot * L::kRow)[w * G + g];
        vw[g] = reinterpret_cast<const uint32_t*>(block + L::kHalf + slot * L::kRow)[w * G + g];
        kp[g] = reinterpret_cast<const uint32_t*>(block + L::kPar + slot * L::kParRow)[g];
        vp[g] = reinterpret_cast<const uint32_t*>(block + L::kHalf + L::kPar + slot * L::kParRow)[g];
      }
    }
  }
  const int64_t at = (static_cast<int64_t>(blockIdx.x) * p.count + i) * D + w * 8;
#pragma unroll
  for (int g = 0; g < G; ++g) {
    ptx::st_global_v4(static_cast<uint16_t*>(p.k) + at + g * 64, values<FMT>(kw[g], kp[g]));
    ptx::st_global_v4(static_cast<uint16_t*>(p.v) + at + g * 64, values<FMT>(vw[g], vp[g]));
  }
}

// ------------------------------------------------------------- evict -------------------------------------------------------------

constexpr int kMostTokens = 1 << 30;
constexpr int kPickThreads = 1024, kPickItems = 4, kPickStretch = kPickThreads * kPickItems;

struct EvictParams {
  const float* weights;          // [B, Hk, S]
  float* out_weights;            // [B, Hk, S_out]: may be `weights`
  const int* lens;
  int *kept, *out_lens;          // [B, Hk, keep], [B]
  uint8_t* cache;
  const int *table, *out_table;
  int B, Hk, S, S_out, keep, recent, sinks, max_pages, out_pages, pages;
  bool in_place;
  uint32_t* status;
};

// Weights as whole numbers in the same order: -0 equals 0, a NaN comes before all others.
CATCOC_DEVICE uint32_t order_key(float w) {
  if (w != w) return 0u;
  const uint32_t u = __float_as_uint(w + 0.0f);
  return (u >> 31) ? ~u : (u | 0x80000000u);
}

// Sum over the block of `x` up to and with this thread, and the whole
CATCOC_DEVICE uint32_t block_scan(uint32_t x, uint32_t* warp_sums, uint32_t& total) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  uint32_t v = x;
#pragma unroll
  for (int o = 1; o < 32; o *= 2) {
    const uint32_t y = __shfl_up_sync(0xffffffffu, v, o);
    if (lane >= o) v += y;
  }
  __syncthreads();
  if (lane == 31) warp_sums[warp] = v;
  __syncthreads();
  uint32_t s = warp_sums[lane];
#pragma unroll
  for (int o = 1; o < 32; o *= 2) {
    const uint32_t y = __shfl_up_sync(0xffffffffu, s, o);
    if (lane >= o) s += y;
  }
  total = __shfl_sync(0xffffffffu, s, 31);
  const uint32_t before = __shfl_sync(0xffffffffu, s, max(warp - 1, 0));
  return v + (warp > 0 ? before : 0u);
}

// Moves the rows of the kept tokens [0, n) of a head to the first places, in stretches: this block's are `first`, `first + step`, ...
// In place one block walks them all: a token never moves up, so the rows of later stretches lie behind all that was written, and
// only the loads and the stores of one stretch need a barrier between them.
template <int D, int THREADS>
struct Move {
  using L = Block<D>;
  static constexpr int kLanes = 2 * L::kRow / 16;           // lanes of a row: its 16-byte pieces, K's then V's
  static constexpr int kUnroll = 4, kRows = THREADS / kLanes * kUnroll, kPars = 2 * kRows / THREADS;

  CATCOC_DEVICE static void run(const EvictParams& p, int bh, int n, int first, int step) {
    const int b = bh / p.Hk, h = bh - b * p.Hk;
    const int* kept = p.kept + static_cast<int64_t>(bh) * p.keep;
    // offsets of the block that token `src` lies in and of the one that it goes to; false: nothing to do
    auto places = [&](int i, int& src, int64_t& from, int64_t& to) {
      if (i >= n) return false;
      src = kept[i];
      if (p.in_place && src == i) return false;
      const int sp = page_of(p.table, static_cast<int64_t>(b) * p.max_pages, src / kPage, p.pages, p.status);
      const int dp = page_of(p.out_table, static_cast<int64_t>(b) * p.out_pages, i / kPage, p.pages, p.status);
      from = (static_cast<int64_t>(sp) * p.Hk + h) * L::kBytes;
      to = (static_cast<int64_t>(dp) * p.Hk + h) * L::kBytes;
      return sp >= 0 && dp >= 0;
    };
    const int sub = threadIdx.x % kLanes;
    const int piece = sub < kLanes / 2 ? sub * 16 : L::kHalf + (sub - kLanes / 2) * 16;
    for (int base = first; base < n; base += step) {
      uint4 x[kUnroll];
      uint2 y[kPars];
      uint8_t *to[kUnroll], *par_to[kPars];
#pragma unroll
      for (int u = 0; u < kUnroll; ++u) {
        const int i = base + u * (kRows / kUnroll) + threadIdx.x / kLanes;
        int src;
        int64_t from, dst;
        to[u] = nullptr;
        if (places(i, src, from, dst)) {
          x[u] = *reinterpret_cast<const uint4*>(p.cache + from + (src % kPage) * L::kRow + piece);
          to[u] = p.cache + dst + (i % kPage) * L::kRow + piece;
        }
      }
#pragma unroll
      for (int u = 0; u < kPars; ++u) {
        const int item = u * THREADS + threadIdx.x, i = base + item / 2, half = (item & 1) * L::kHalf + L::kPar;
        int src;
        int64_t from, dst;
        par_to[u] = nullptr;
        if (places(i, src, from, dst)) {
          const uint8_t* at = p.cache + from + half + (src % kPage) * L::kParRow;
          if constexpr (L::kParRow == 8) y[u] = *reinterpret_cast<const uint2*>(at);
          else y[u].x = *reinterpret_cast<const uint32_t*>(at);
          par_to[u] = p.cache + dst + half + (i % kPage) * L::kParRow;
        }
      }
      if (p.in_place) __syncthreads();
#pragma unroll
      for (int u = 0; u < kUnroll; ++u)
        if (to[u] != nullptr) *reinterpret_cast<uint4*>(to[u]) = x[u];
#pragma unroll
      for (int u = 0; u < kPars; ++u) {
        if (par_to[u] == nullptr) continue;
        if constexpr (L::kParRow == 8) *reinterpret_cast<uint2*>(par_to[u]) = y[u];
        else *reinterpret_cast<uint32_t*>(par_to[u]) = y[u].x;
      }
    }
  }
};

// One CTA per (sequence, head). The weight of the last token that stays is found 11 bits at a time, from the top: a histogram of
// these bits over the tokens that agree with what is found so far. Then all tokens pass once more in order; those above it
// stay, and of those equal to it the first ones. MOVE: the CTA moves the tokens too.
template <int D, bool MOVE>
__global__ void __launch_bounds__(kPickThreads) kv4_evict_kernel(const EvictParams p) {
  __shared__ uint32_t hist[2048], warp_sums[32], found[2];
  ptx::grid_dependency_wait();
  if constexpr (!MOVE) ptx::launch_dependents();
  const int bh = blockIdx.x, b = bh / p.Hk, tid = threadIdx.x;
  const int n = seq_len(p.lens, b, p.max_pages * kPage, p.status);
  const int stay = min(n, p.keep);
  const float* w = p.weights + static_cast<int64_t>(bh) * p.S;
  float* ow = p.out_weights + static_cast<int64_t>(bh) * p.S_out;
  int* kept = p.kept + static_cast<int64_t>(bh) * p.keep;
  if (bh == b * p.Hk && tid == 0) p.out_lens[b] = stay;
  const bool all = n <= p.keep;
  // (sinks + recent <= keep < n, so the two ends do not meet)
  const int c0 = all ? 0 : p.sinks, c1 = all ? 0 : n - p.recent;                 // the candidates
  uint32_t need = all ? 0u : static_cast<uint32_t>(p.keep - p.sinks - p.recent);   // of them stay
  const bool some = need > 0u;
  // four tokens in a row a thread; a sequence of one stretch stays in the registers
  float x[kPickItems];
  auto load = [&](int base) {
#pragma unroll
    for (int e = 0; e < kPickItems; ++e) {
      const int i = base + tid * kPickItems + e;
      x[e] = i < n ? w[i] : 0.0f;
    }
  };
  load(0);
  uint32_t key = 0u;
  if (some) {
#pragma unroll 1
    for (int shift = 21; shift >= 0; shift = shift == 21 ? 10 : shift - 10) {
      const uint32_t mask = shift == 0 ? 1023u : 2047u;
      hist[tid] = hist[tid + 1024] = 0u;
      __syncthreads();
      for (int base = 0; base < n; base += kPickStretch) {
        if (n > kPickStretch) load(base);
#pragma unroll
        for (int e = 0; e < kPickItems; ++e) {
          const int i = base + tid * kPickItems + e;
          const uint32_t k = order_key(x[e]);
          const bool agrees = shift == 21 || (shift == 10 ? (k ^ key) >> 21 : (k ^ key) >> 10) == 0u;
          if (i >= c0 && i < c1 && agrees) atomicAdd(&hist[(k >> shift) & mask], 1u);
        }
      }
      __syncthreads();
      // the bin in which the need-th largest lies: thread i looks at the bins 2047 - 2 i and 2046 - 2 i
      const uint32_t top = hist[2047 - 2 * tid], next = hist[2046 - 2 * tid];
      uint32_t total;
      const uint32_t upto = block_scan(top + next, warp_sums, total), above = upto - top - next;
      if (upto >= need && above < need) {
        const bool first = above + top >= need;
        found[0] = static_cast<uint32_t>(2047 - 2 * tid) - (first ? 0u : 1u);
        found[1] = need - above - (first ? 0u : top);
      }
      __syncthreads();
      key |= found[0] << shift;
      need = found[1];
    }
  }
  // `need` of the tokens whose weight is the key itself stay, the first ones
  uint32_t above = 0u, equals = 0u;                  // tokens before this stretch that stay for their place or weight, and equal ones
  for (int base = 0; base < n; base += kPickStretch) {
    if (n > kPickStretch) load(base);
    uint32_t up = 0u, eq = 0u;                       // the same of this thread's, a bit each
#pragma unroll
    for (int e = 0; e < kPickItems; ++e) {
      const int i = base + tid * kPickItems + e;
      const uint32_t k = order_key(x[e]);
      const bool candidate = i >= c0 && i < c1;
      if (i < n && (!candidate || (some && k > key))) up |= 1u << e;
      if (candidate && some && k == key) eq |= 1u << e;
    }
    // (both counts of a stretch fit 16 bits)
    uint32_t total;
    const uint32_t mine = __popc(up) | (__popc(eq) << 16), upto = block_scan(mine, warp_sums, total) - mine;
    uint32_t a = above + (upto & 0xffffu), q = equals + (upto >> 16);
    // (the scan's barriers stand between the loads of this stretch and its stores, which land at or before it)
#pragma unroll
    for (int e = 0; e < kPickItems; ++e) {
      const bool is_up = (up >> e) & 1u, is_eq = (eq >> e) & 1u;
      if (is_up || (is_eq && q < need)) {
        const uint32_t at = a + min(q, need);
        kept[at] = base + tid * kPickItems + e;
        ow[at] = x[e];
      }
      a += is_up;
      q += is_eq;
    }
    above += total & 0xffffu;
    equals += total >> 16;
  }
  __syncthreads();
  for (int i = stay + tid; i < p.keep; i += kPickThreads) kept[i] = -1;
  for (int i = stay + tid; i < p.S_out; i += kPickThreads) ow[i] = 0.0f;
  if constexpr (MOVE) {
    using M = Move<D, kPickThreads>;
    if (!(p.in_place && all)) M::run(p, bh, stay, 0, M::kRows);
  }
}

// The moves of a head dealt out over grid y, into other pages than the sequence's own
constexpr int kMoveThreads = 256;
template <int D>
__global__ void __launch_bounds__(kMoveThreads) kv4_move_kernel(const EvictParams p) {
  using M = Move<D, kMoveThreads>;
  ptx::grid_dependency_wait();
  M::run(p, blockIdx.x, p.out_lens[blockIdx.x / p.Hk], blockIdx.y * M::kRows, gridDim.y * M::kRows);
}

int bad(const char* what) {
  set_error("%s", what);
  return CATCOC_E_BAD_ARG;
}

}  // namespace

extern "C" int64_t catcoc_kv4_block_bytes(int D) { return D == 128 ? Block<128>::kBytes : D == 64 ? Block<64>::kBytes : -1; }

namespace {
// What all calls share; `types`: fp16 and bf16 are told apart
int common(const CatcocKv4Call* c, const char* what, bool types) {
  if (!c || c->B <= 0 || c->Hk <= 0 || c->pages <= 0 || c->max_pages <= 0) { set_error("%s: bad arguments", what); return CATCOC_E_BAD_ARG; }
  if (c->D != 64 && c->D != 128) { set_error("%s: head dimension %d (64 and 128 are built)", what, c->D); return CATCOC_E_UNSUPPORTED; }
  if (types && c->fmt != CATCOC_FMT_F16 && c->fmt != CATCOC_FMT_BF16) { set_error("%s takes fp16 / bf16", what); return CATCOC_E_UNSUPPORTED; }
  if (static_cast<int64_t>(c->B) * c->Hk > 0x7fffffff || static_cast<int64_t>(c->max_pages) * kPage > 0x7fffffff) { set_error("%s: too many tokens", what); return CATCOC_E_TOO_LARGE; }
  return CATCOC_OK;
}
bool unaligned(const void* a, const void* b = nullptr, const void* c = nullptr) {
  return ((reinterpret_cast<uintptr_t>(a) | reinterpret_cast<uintptr_t>(b) | reinterpret_cast<uintptr_t>(c)) & 15) != 0;
}
}  // namespace

extern "C" int catcoc_kv4_append(const CatcocKv4Call* c, void* cache, const void* k, const void* v, const int* block_table, const int* kv_lens,
                                 const int* ends, uint32_t* status, void* stream) {
  const int rc = common(c, "kv4_append", true);
  if (rc != CATCOC_OK) return rc;
  if (!cache || !k || !v || !block_table || !kv_lens || !status || c->T <= 0 || (!ends && c->T % c->B)) return bad("kv4_append: bad arguments");
  if (unaligned(cache, k, v) || ((c->k_token | c->k_head | c->v_token | c->v_head) & 7)) {
    set_error("kv4_append: rows must begin at 16-byte boundaries");
    return CATCOC_E_ALIGNMENT;
  }
  const int64_t blocks = (static_cast<int64_t>(c->T) * c->Hk * (c->D / 16) + 255) / 256;
  if (blocks > 0x7fffffff) { set_error("kv4_append: too many tokens"); return CATCOC_E_TOO_LARGE; }
  const AppendParams p{k, v, c->k_token, c->k_head, c->v_token, c->v_head, static_cast<uint8_t*>(cache), block_table, kv_lens, ends,
                       c->T, c->B, c->Hk, ends ? 1 : c->T / c->B, c->max_pages, c->pages, status};
  auto launch = [&](auto kernel) -> int {
    CATCOC_CUDA_OK(launch_overlapped(kernel, dim3(static_cast<unsigned>(blocks)), dim3(256), 0, static_cast<cudaStream_t>(stream), p));
    return CATCOC_OK;
  };
  if (c->D == 128) return c->fmt == CATCOC_FMT_BF16 ? launch(kv4_append_kernel<128, FMT_BF16>) : launch(kv4_append_kernel<128, FMT_F16>);
  return c->fmt == CATCOC_FMT_BF16 ? launch(kv4_append_kernel<64, FMT_BF16>) : launch(kv4_append_kernel<64, FMT_F16>);
}

extern "C" int catcoc_kv4_read(const CatcocKv4Call* c, const void* cache, const int* block_table, const int* kv_lens, const int* start, void* k, void* v,
                               uint32_t* status, void* stream) {
  const int rc = common(c, "kv4_read", true);
  if (rc != CATCOC_OK) return rc;
  if (!cache || !block_table || !kv_lens || !k || !v || !status || c->count <= 0) return bad("kv4_read: bad arguments");
  if (unaligned(cache, k, v)) { set_error("kv4_read: buffers must be 16-byte aligned"); return CATCOC_E_ALIGNMENT; }
  const int64_t heads = static_cast<int64_t>(c->B) * c->Hk, chunks = (static_cast<int64_t>(c->count) + 31) / 32;
  if (chunks > 65535) { set_error("kv4_read: too many tokens"); return CATCOC_E_TOO_LARGE; }
  const ReadParams p{static_cast<const uint8_t*>(cache), block_table, kv_lens, start, k, v, c->B, c->Hk, c->count, c->max_pages, c->pages, status};
  auto launch = [&](auto kernel) -> int {
    CATCOC_CUDA_OK(launch_overlapped(kernel, dim3(static_cast<unsigned>(heads), static_cast<unsigned>(chunks)), dim3(256), 0, static_cast<cudaStream_t>(stream), p));
    return CATCOC_OK;
  };
  if (c->D == 128) return c->fmt == CATCOC_FMT_BF16 ? launch(kv4_read_kernel<128, FMT_BF16>) : launch(kv4_read_kernel<128, FMT_F16>);
  return c->fmt == CATCOC_FMT_BF16 ? launch(kv4_read_kernel<64, FMT_BF16>) : launch(kv4_read_kernel<64, FMT_F16>);
}

extern "C" int catcoc_kv4_evict(const CatcocKv4Call* c, void* cache, const float* weights, float* out_weights, const int* block_table, const int* out_table,
                                const int* kv_lens, int* kept, int* out_lens, uint32_t* status, void* stream_) {
  const int rc = common(c, "kv4_evict", false);
  if (rc != CATCOC_OK) return rc;
  if (!cache || !weights || !out_weights || !block_table || !out_table || !kv_lens || !kept || !out_lens || !status || c->out_pages <= 0 || c->keep <= 0 ||
      c->recent < 0 || c->sinks < 0)
    return bad("kv4_evict: bad arguments");
  const int64_t capacity = static_cast<int64_t>(c->max_pages) * kPage, heads = static_cast<int64_t>(c->B) * c->Hk;
  if (static_cast<int64_t>(c->recent) + c->sinks > c->keep) return bad("kv4_evict: the first and the last tokens are more than what is kept");
  // (the kernel steps over tokens, places and weights in int, 4096 and more at a time)
  if (c->keep > kMostTokens || capacity > kMostTokens || c->S_out > kMostTokens) { set_error("kv4_evict: more than 2^30 tokens"); return CATCOC_E_TOO_LARGE; }
  const int64_t most = std::min<int64_t>(c->keep, capacity);      // tokens that can stay
  if (c->S < capacity || static_cast<int64_t>(c->out_pages) * kPage < most || c->S_out < most) return bad("kv4_evict: the weights or the new pages are too short");
  if (unaligned(cache)) { set_error("kv4_evict: the cache must be 16-byte aligned"); return CATCOC_E_ALIGNMENT; }
  cudaStream_t stream = static_cast<cudaStream_t>(stream_);
  const bool in_place = out_table == block_table;
  const EvictParams p{weights, out_weights, kv_lens, kept, out_lens, static_cast<uint8_t*>(cache), block_table, out_table, c->B, c->Hk, c->S, c->S_out,
                      c->keep, c->recent, c->sinks, c->max_pages, c->out_pages, c->pages, in_place, status};
  auto launch = [&](auto kernel, dim3 grid, int threads) -> int {
    CATCOC_CUDA_OK(launch_overlapped(kernel, grid, dim3(static_cast<unsigned>(threads)), 0, stream, p));
    return CATCOC_OK;
  };
  // One launch where the heads fill half of the SMs or have little to move, and in place, where a head's moves are in order anyway.
  const dim3 grid(static_cast<unsigned>(heads));
  int device = 0;
  cudaGetDevice(&device);
  if (in_place || 2 * heads >= catcoc_num_sms(device) || most <= 1024)
    return c->D == 128 ? launch(kv4_evict_kernel<128, true>, grid, kPickThreads) : launch(kv4_evict_kernel<64, true>, grid, kPickThreads);
  const int first = c->D == 128 ? launch(kv4_evict_kernel<128, false>, grid, kPickThreads) : launch(kv4_evict_kernel<64, false>, grid, kPickThreads);
  if (first != CATCOC_OK) return first;
  const int rows = c->D == 128 ? Move<128, kMoveThreads>::kRows : Move<64, kMoveThreads>::kRows;
  const dim3 dealt(static_cast<unsigned>(heads), static_cast<unsigned>(std::min<int64_t>(1024, (most + rows - 1) / rows)));
  return c->D == 128 ? launch(kv4_move_kernel<128>, dealt, kMoveThreads) : launch(kv4_move_kernel<64>, dealt, kMoveThreads);
}
