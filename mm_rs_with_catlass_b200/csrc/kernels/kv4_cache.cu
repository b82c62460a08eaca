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
CATCOC_DEVICE void unpack8(uint4 a, float (&f)[8]) {
  const uint32_t u[4] = {a.x, a.y, a.z, a.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if constexpr (FMT == FMT_BF16) {
      f[2 * i] = bf16_lo(u[i]);
      f[2 * i + 1] = bf16_hi(u[i]);
    } else {
      const float2 v = __half22float2(*reinterpret_cast<const __half2*>(&u[i]));
      f[2 * i] = v.x;
      f[2 * i + 1] = v.y;
    }
  }
}

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

// Codes of eight channels and the parameters of their group, whose other 56 channels are in the lanes `lane ^ G, 2 G, 4 G` ...
template <int FMT, int G>
CATCOC_DEVICE uint32_t quantise(uint4 raw, uint32_t& param) {
  float f[8];
  unpack8<FMT>(raw, f);
  float lo = f[0], hi = f[0];
  // a value that is no number, or an infinity, makes the group's parameters NaN (x * 0 is NaN for both)
  float odd = f[0] * 0.0f;
#pragma unroll
  for (int i = 1; i < 8; ++i) {
    lo = fminf(lo, f[i]);
    hi = fmaxf(hi, f[i]);
    odd += f[i] * 0.0f;
  }
#pragma unroll
  for (int o = G; o < 8 * G; o *= 2) {
    lo = fminf(lo, __shfl_xor_sync(0xffffffffu, lo, o));
    hi = fmaxf(hi, __shfl_xor_sync(0xffffffffu, hi, o));
    odd += __shfl_xor_sync(0xffffffffu, odd, o);
  }
  // each rounding is the cache's own: the scale and the zero are held in bf16, and the codes are taken against the rounded ones
  float s = __bfloat162float(__float2bfloat16_rn((hi - lo) * (1.0f / 15.0f)));
  const float z = __bfloat162float(__float2bfloat16_rn(lo));
  if (s < 1.17549435e-38f) s = 0.0f;                   // a group of one value, or a range whose reciprocal would overflow
  if (!(odd == 0.0f) || !(s <= 3.4e38f)) s = __uint_as_float(0x7fc00000u);
  const float r = s > 0.0f ? 1.0f / s : 0.0f;
  uint32_t word = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const int c = min(15, max(0, __float2int_rn(__fmul_rn(__fsub_rn(f[i], z), r))));
    word |= static_cast<uint32_t>(c) << (4 * i);
  }
  param = (__float_as_uint(s) >> 16) | (__float_as_uint(z) & 0xffff0000u);
  return word;
}

// A thread: eight channels of K and of V of one token and head. 8 G lanes make a row and leave its words in order.
template <int D, int FMT>
__global__ void __launch_bounds__(256) kv4_append_kernel(const AppendParams p) {
  using L = Block<D>;
  constexpr int G = L::kGroups, kLanes = 8 * G;
  ptx::grid_dependency_wait();
  const int lane = threadIdx.x & 31;
  const int64_t idx = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x;
  const int64_t rows = static_cast<int64_t>(p.T) * p.Hk;
  const int64_t row = idx / kLanes;
  const int j = static_cast<int>(idx % kLanes), g = j % G, w = j / G;
  const bool real = row < rows;
  const int t = real ? static_cast<int>(row / p.Hk) : p.T, h = real ? static_cast<int>(row - static_cast<int64_t>(t) * p.Hk) : 0;
  uint4 kr = make_uint4(0, 0, 0, 0), vr = kr;
  if (real) {
    const int c = g * 64 + w * 8;
    kr = *reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(p.k) + t * p.k_token + h * p.k_head + c);
    vr = *reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(p.v) + t * p.v_token + h * p.v_head + c);
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
      if (n < 32 && behind == 0) behind = mine == 0x7fffffff ? -1 : mine - t;
      if (behind == 0) b += 32;
      else if (n < 32 && b == base) b = base + n;
    }
  }
  uint32_t kp, vp;
  const uint32_t kw = quantise<FMT, G>(kr, kp), vw = quantise<FMT, G>(vr, vp);
  if (!real || b >= p.B || behind <= 0) return;           // a token behind the last sequence
  const int len = seq_len(p.lens, b, p.max_pages * kPage, p.status);
  const int pos = len - behind;
  if (pos < 0) { if (j == 0) note(p.status, kErrLen, len, behind); return; }
  const int page = page_of(p.table, static_cast<int64_t>(b) * p.max_pages, pos / kPage, p.pages, p.status);
  if (page < 0) return;
  uint8_t* block = p.cache + (static_cast<int64_t>(page) * p.Hk + h) * L::kBytes;
  const int slot = pos % kPage;
  *reinterpret_cast<uint32_t*>(block + slot * L::kRow + j * 4) = kw;
  *reinterpret_cast<uint32_t*>(block + L::kHalf + slot * L::kRow + j * 4) = vw;
  if (w == 0) *reinterpret_cast<uint32_t*>(block + L::kPar + slot * L::kParRow + g * 4) = kp;
  if (w == 1) *reinterpret_cast<uint32_t*>(block + L::kHalf + L::kPar + slot * L::kParRow + g * 4) = vp;
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

constexpr int kPickThreads = 1024;

struct PickParams {
  const float* weights;          // [B, Hk, S]
  float* out_weights;            // [B, Hk, S_out]: may be `weights`
  const int* lens;
  int *kept, *out_lens;          // [B, Hk, keep], [B]
  int B, Hk, S, S_out, keep, recent, sinks, capacity;
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

// One CTA per (sequence, head). The weight of the last token that stays is found a byte at a time, from the top: a histogram of the
// byte over the tokens that agree with what is found so far. Then all tokens pass once more in order; those above it stay,
// and of those equal to it the first ones.
__global__ void __launch_bounds__(kPickThreads) kv4_pick_kernel(const PickParams p) {
  __shared__ uint32_t hist[256], warp_sums[32], found[2];
  ptx::grid_dependency_wait();
  ptx::launch_dependents();
  const int bh = blockIdx.x, b = bh / p.Hk, tid = threadIdx.x;
  const int n = seq_len(p.lens, b, p.capacity, p.status);
  const int stay = min(n, p.keep);
  const float* w = p.weights + static_cast<int64_t>(bh) * p.S;
  float* ow = p.out_weights + static_cast<int64_t>(bh) * p.S_out;
  int* kept = p.kept + static_cast<int64_t>(bh) * p.keep;
  if (bh == b * p.Hk && tid == 0) p.out_lens[b] = stay;
  const bool all = n <= p.keep;
  // (sinks + recent <= keep < n, so the two ends do not meet)
  const int c0 = all ? 0 : p.sinks, c1 = all ? n : n - p.recent;
  uint32_t need = all ? 0u : static_cast<uint32_t>(p.keep - p.sinks - p.recent);   // of the candidates [c0, c1)
  uint32_t key = 0u;
  if (need > 0u) {
    for (int shift = 24; shift >= 0; shift -= 8) {
      for (int i = tid; i < 256; i += kPickThreads) hist[i] = 0u;
      __syncthreads();
      for (int i = c0 + tid; i < c1; i += kPickThreads) {
        const uint32_t k = order_key(w[i]);
        if (shift == 24 || (k >> (shift + 8)) == (key >> (shift + 8))) atomicAdd(&hist[(k >> shift) & 255u], 1u);
      }
      __syncthreads();
      // the byte in whose bin the need-th largest lies: thread i looks at bin 255 - i
      const uint32_t mine = tid < 256 ? hist[255 - tid] : 0u;
      uint32_t total;
      const uint32_t upto = block_scan(mine, warp_sums, total);
      if (tid < 256 && upto >= need && upto - mine < need) {
        found[0] = static_cast<uint32_t>(255 - tid);
        found[1] = need - (upto - mine);
      }
      __syncthreads();
      key |= found[0] << shift;
      need = found[1];
      __syncthreads();
    }
  }
  // `need` of the tokens whose weight is the key itself stay, the first ones
  uint32_t placed = 0u, equals = 0u;
  for (int base = 0; base < n; base += kPickThreads) {
    const int i = base + tid;
    const bool in = i < n, candidate = !all && in && i >= c0 && i < c1;
    const float x = in ? w[i] : 0.0f;
    const uint32_t k = order_key(x);
    const bool equal = candidate && p.keep > p.sinks + p.recent && k == key;
    uint32_t eq_total, total;
    const uint32_t eq = block_scan(equal ? 1u : 0u, warp_sums, eq_total);
    const bool stays = in && (!candidate || (p.keep > p.sinks + p.recent && (k > key || (equal && equals + eq <= need))));
    const uint32_t at = block_scan(stays ? 1u : 0u, warp_sums, total);
    // (the scans' barriers stand between the loads of this stretch and its stores, which land at or before it)
    if (stays) {
      kept[placed + at - 1] = i;
      ow[placed + at - 1] = x;
    }
    placed += total;
    equals += eq_total;
  }
  __syncthreads();
  for (int i = stay + tid; i < p.keep; i += kPickThreads) kept[i] = -1;
  for (int i = stay + tid; i < p.S_out; i += kPickThreads) ow[i] = 0.0f;
}

struct MoveParams {
  uint8_t* cache;
  const int *table, *out_table, *kept, *lens;    // lens: the new lengths
  int B, Hk, keep, max_pages, out_pages, pages;
  bool in_place;
  uint32_t* status;
};

constexpr int kMoveThreads = 256;

// The kept tokens' rows go to the first places, in order. One CTA per (sequence, head, K or V) walks them in stretches when
// the places are the sequence's own pages: a token never moves up, so the rows of later stretches lie behind all that was
// written, and only the loads and the stores of one stretch need a barrier between them. Into other pages the stretches are
// dealt out over grid z.
template <int D>
__global__ void __launch_bounds__(kMoveThreads) kv4_move_kernel(const MoveParams p) {
  using L = Block<D>;
  constexpr int kPieces = L::kRow / 16;                  // 16-byte pieces of a row's codes; thread `kPieces` takes the parameters
  constexpr int kRows = 4 * kMoveThreads / 8;            // rows of a stretch: 8 threads a row, 4 rows a thread
  ptx::grid_dependency_wait();
  const int bh = blockIdx.x, b = bh / p.Hk, h = bh - b * p.Hk;
  const int n = p.lens[b];
  const int* kept = p.kept + static_cast<int64_t>(bh) * p.keep;
  const int sub = threadIdx.x & 7, half = blockIdx.y * L::kHalf;
  for (int base = blockIdx.z * kRows; base < n; base += gridDim.z * kRows) {
    uint4 x[4];
    uint8_t* to[4];
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const int i = base + u * (kRows / 4) + (threadIdx.x >> 3);
      to[u] = nullptr;
      if (i < n && sub <= kPieces) {
        const int src = kept[i];
        const int sp = page_of(p.table, static_cast<int64_t>(b) * p.max_pages, src / kPage, p.pages, p.status);
        const int dp = page_of(p.out_table, static_cast<int64_t>(b) * p.out_pages, i / kPage, p.pages, p.status);
        if (sp >= 0 && dp >= 0 && !(p.in_place && src == i)) {
          const uint8_t* from = p.cache + (static_cast<int64_t>(sp) * p.Hk + h) * L::kBytes + half;
          uint8_t* dst = p.cache + (static_cast<int64_t>(dp) * p.Hk + h) * L::kBytes + half;
          if (sub < kPieces) {
            x[u] = *reinterpret_cast<const uint4*>(from + (src % kPage) * L::kRow + sub * 16);
            to[u] = dst + (i % kPage) * L::kRow + sub * 16;
          } else {
            if constexpr (L::kParRow == 8) *reinterpret_cast<uint2*>(&x[u]) = *reinterpret_cast<const uint2*>(from + L::kPar + (src % kPage) * 8);
            else x[u].x = *reinterpret_cast<const uint32_t*>(from + L::kPar + (src % kPage) * 4);
            to[u] = dst + L::kPar + (i % kPage) * L::kParRow;
          }
        }
      }
    }
    if (p.in_place) __syncthreads();
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      if (to[u] == nullptr) continue;
      if (sub < kPieces) *reinterpret_cast<uint4*>(to[u]) = x[u];
      else if constexpr (L::kParRow == 8) *reinterpret_cast<uint2*>(to[u]) = make_uint2(x[u].x, x[u].y);
      else *reinterpret_cast<uint32_t*>(to[u]) = x[u].x;
    }
  }
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
  const int64_t blocks = (static_cast<int64_t>(c->T) * c->Hk * (c->D / 8) + 255) / 256;
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
  const int64_t most = std::min<int64_t>(c->keep, capacity);      // tokens that can stay
  if (c->S < capacity || static_cast<int64_t>(c->out_pages) * kPage < most || c->S_out < most) return bad("kv4_evict: the weights or the new pages are too short");
  if (unaligned(cache)) { set_error("kv4_evict: the cache must be 16-byte aligned"); return CATCOC_E_ALIGNMENT; }
  cudaStream_t stream = static_cast<cudaStream_t>(stream_);
  const bool in_place = out_table == block_table;
  const PickParams pick{weights, out_weights, kv_lens, kept, out_lens, c->B, c->Hk, c->S, c->S_out, c->keep, c->recent, c->sinks, static_cast<int>(capacity), status};
  CATCOC_CUDA_OK(launch_overlapped(kv4_pick_kernel, dim3(static_cast<unsigned>(heads)), dim3(kPickThreads), 0, stream, pick));
  const MoveParams move{static_cast<uint8_t*>(cache), block_table, out_table, kept, out_lens, c->B, c->Hk, c->keep, c->max_pages, c->out_pages, c->pages, in_place, status};
  const unsigned stretches = in_place ? 1u : static_cast<unsigned>(std::min<int64_t>(64, (most + 127) / 128));
  auto launch = [&](auto kernel) -> int {
    CATCOC_CUDA_OK(launch_overlapped(kernel, dim3(static_cast<unsigned>(heads), 2u, stretches), dim3(kMoveThreads), 0, stream, move));
    return CATCOC_OK;
  };
  return c->D == 128 ? launch(kv4_move_kernel<128>) : launch(kv4_move_kernel<64>);
}
