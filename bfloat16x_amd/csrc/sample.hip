// Token sampling (include/bf16x_llama.h): temperature, top-k, top-p and min-p
// from given uniform numbers.
//
// All three filters keep a prefix of the row's tokens in the order (larger
// logit, then lower index), so the kept set is one threshold in that order: of
// the 64-bit number (the logit's bits in ascending order, then the complement of
// the index), which is different for every token.  It is found without sorting
// the row: the weights of a row span 32 nepers at most (smaller ones round to
// nothing in 2^-44), which are cut into kBins bins; counts and masses per bin
// tell the bin (for top-p behind top-k, the few bins) that holds the threshold,
// and only the tokens of those are sorted.  The steps, one launch each, chunks
// of a row in parallel:
//   1. largest and smallest logit of every chunk;
//   2. count and mass of the bins (rows with top-k or top-p), or the mass of
//      every chunk (rows without);
//   3. the bins of the threshold; their tokens to a list; the mass of every
//      chunk in the bins above (rows with top-k or top-p);
//   4. one workgroup per row: the list sorted, the threshold, the chunk in which
//      the running mass passes u, the token.
// Masses are integers of 2^-44 of the largest weight: their sums are the same in
// any order, so atomics do not change results, and two neighbouring tokens'
// border moves by 1e-11 of the total at most, where an fp32 sum would move it by
// the probability of an unlikely token.  The exponential is a Taylor polynomial
// of degree 11 in fp64 (relative error 1e-14 on half an octave).
#include "bf16x_device.h"
#include "launch_common.h"
#include "../../include/bf16x_llama.h"

namespace {
using namespace bf16x;

typedef float f4 __attribute__((ext_vector_type(4)));
typedef unsigned long long u64;

constexpr int kBins = 1024;
constexpr int kList = 4096;               // tokens of the threshold's bins that step 4 sorts in LDS
constexpr int kMaxChunks = 256;
constexpr int kT = 256;                   // threads of steps 1 to 3
constexpr int kDrawT = 1024;              // threads of step 4
constexpr double kSpan = 32.0;            // nepers; exp(-32) < 2^-46
constexpr int64_t kMaxVocab = (int64_t)1 << 20;

// What steps 3 and 4 know of the bins of a row.
struct Cut {
  uint32_t k_bin, p_first, p_last, sure;  // top-k's bin, top-p's bins, bins surely kept (all below `sure`); ~0: none
  uint32_t before_k;                      // tokens in the bins before top-k's
  uint32_t in_k;                          // tokens in it
  u64 mass_k;                             // mass of the bins before top-k's (no top-k: of all)
  u64 mass_p;                             // mass of the bins before top-p's first
};

struct SampleArgs {
  const void* logits;
  int64_t stride;
  int vocab, chunk, chunks;
  const float* u;
  int64_t n_u;
  bf16x_sample_settings s;
  int64_t* token;
  float* logprob;
  int32_t* state;
  int32_t* history;
  int64_t history_len;
  float *cmax, *cmin;                     // [rows][chunks]
  int32_t* cidx;                          // [rows][chunks] first index of the chunk's maximum
  u64* cmass;                             // [rows][chunks]
  u64* hmass;                             // [rows][kBins]
  uint32_t* hcount;                       // [rows][kBins]
  uint32_t* listed;                       // [rows] tokens put into the list (more than kList: the list is not whole)
  Cut* cut;                               // [rows]
  u64* list;                              // [rows][kList]
};

struct Setting {
  double inv_t;                           // 0 where T is not above 0
  bool greedy, k_on, p_on;
  uint32_t k;
  double p, min_p;
};

__device__ __forceinline__ Setting setting_of(const SampleArgs& a, int row) {
  const float t = a.s.temperature ? a.s.temperature[row] : a.s.temperature_all;
  const int32_t k = a.s.top_k ? a.s.top_k[row] : a.s.top_k_all;
  const float p = a.s.top_p ? a.s.top_p[row] : a.s.top_p_all;
  const float q = a.s.min_p ? a.s.min_p[row] : a.s.min_p_all;
  Setting s;
  s.greedy = !(t > 0.f);
  s.inv_t = s.greedy ? 0.0 : 1.0 / (double)t;
  s.k_on = !s.greedy && k > 0 && k < a.vocab;
  s.k = (uint32_t)k;
  s.p_on = !s.greedy && p < 1.f;
  s.p = p > 0.f ? (double)p : 0.0;
  s.min_p = fminf(q, 1.f);
  return s;
}

// Logits i .. i + 7 (i a multiple of 8) as fp32; -inf for NaN and beyond the row.
template <int TYPE>
__device__ __forceinline__ void logits8(const SampleArgs& a, const void* row, bool vec, int i, float (&x)[8]) {
  if (vec && i + 8 <= a.vocab) {
    if constexpr (TYPE == BF16X_F32) {
      const f4 p = *(const f4*)((const float*)row + i), q = *(const f4*)((const float*)row + i + 4);
#pragma unroll
      for (int e = 0; e < 4; ++e) x[e] = p[e], x[4 + e] = q[e];
    } else {
      const u32x4 r = *(const u32x4*)((const uint16_t*)row + i);
      const uint32_t w[4] = {r.x, r.y, r.z, r.w};
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        if constexpr (TYPE == BF16X_BF16) {
          x[2 * e] = bf16lo_to_f32(w[e]);
          x[2 * e + 1] = bf16hi_to_f32(w[e]);
        } else {
          x[2 * e] = (float)__builtin_bit_cast(_Float16, (uint16_t)w[e]);
          x[2 * e + 1] = (float)__builtin_bit_cast(_Float16, (uint16_t)(w[e] >> 16));
        }
      }
    }
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      float v = -INFINITY;
      if (i + e < a.vocab) {
        if constexpr (TYPE == BF16X_F32) v = ((const float*)row)[i + e];
        else if constexpr (TYPE == BF16X_BF16) v = __uint_as_float((uint32_t)((const uint16_t*)row)[i + e] << 16);
        else v = (float)((const _Float16*)row)[i + e];
      }
      x[e] = v;
    }
  }
#pragma unroll
  for (int e = 0; e < 8; ++e) x[e] = x[e] == x[e] ? x[e] : -INFINITY;
}

template <int TYPE>
__device__ __forceinline__ const void* row_of(const SampleArgs& a, int row, bool& vec) {
  const char* p = (const char*)a.logits + (int64_t)row * a.stride * (TYPE == BF16X_F32 ? 4 : 2);
  vec = ((uintptr_t)p & 15u) == 0;
  return p;
}

// Ascending order of floats as unsigned numbers, and back (-0 and 0 are one value: callers add 0).
__device__ __forceinline__ uint32_t ordered(float x) {
  const uint32_t b = __float_as_uint(x + 0.f);
  return b ^ ((uint32_t)((int32_t)b >> 31) | 0x80000000u);
}
__device__ __forceinline__ float unordered(uint32_t o) {
  return __uint_as_float(o ^ (o >> 31 ? 0x80000000u : 0xFFFFFFFFu));
}
__device__ __forceinline__ u64 place_of(float x, int i) { return (u64)ordered(x) << 32 | (uint32_t)~i; }

// log of the weight of logit x under the row's maximum m: 0 for the maximum
// itself (m may be +inf), something not >= -kSpan for what is never drawn.
__device__ __forceinline__ double log_weight(float x, float m, double inv_t) {
  return x == m ? 0.0 : ((double)x - (double)m) * inv_t;
}

// exp(y) for -kSpan <= y <= 0.
__device__ __forceinline__ double weight_of(double y) {
  const double z = y * 1.4426950408889634074;
  const double n = __builtin_rint(z);
  const double r = (z - n) * 0.69314718055994530942;
  double p = 1.0 / 39916800.0;
  p = fma(p, r, 1.0 / 3628800.0);
  p = fma(p, r, 1.0 / 362880.0);
  p = fma(p, r, 1.0 / 40320.0);
  p = fma(p, r, 1.0 / 5040.0);
  p = fma(p, r, 1.0 / 720.0);
  p = fma(p, r, 1.0 / 120.0);
  p = fma(p, r, 1.0 / 24.0);
  p = fma(p, r, 1.0 / 6.0);
  p = fma(p, r, 0.5);
  p = fma(p, r, 1.0);
  p = fma(p, r, 1.0);
  return p * __longlong_as_double((long long)((int)n + 1023) << 52);
}
// A weight (0 .. 1) as an integer of 2^-44, rounded by the addition of 2^52.
__device__ __forceinline__ u64 mass_of(double w) {
  return (u64)__double_as_longlong(w * 0x1p44 + 0x1p52) & ((1ull << 52) - 1);
}

template <class T>
__device__ __forceinline__ T shfl_up_t(T v, int o) {
  if constexpr (sizeof(T) == 8)
    return (T)((u64)__shfl_up((uint32_t)(v >> 32), o, 64) << 32 | __shfl_up((uint32_t)v, o, 64));
  else
    return __shfl_up(v, o, 64);
}

// Inclusive prefix over the NT threads of a workgroup; `red` holds NT / 64 values.
template <int NT, class T>
__device__ __forceinline__ T block_prefix(T v, T* red, T& total) {
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const T u = shfl_up_t(v, o);
    if (lane >= o) v += u;
  }
  __syncthreads();
  if (lane == 63) red[w] = v;
  __syncthreads();
  T before = 0, all = 0;
#pragma unroll
  for (int k = 0; k < NT / 64; ++k) {
    const T x = red[k];
    if (k < w) before += x;
    all += x;
  }
  total = all;
  return before + v;
}

// The row's maximum, minimum (finite or +inf logits) and first index of the maximum, from its chunks'.
struct Extremes {
  float mx, mn;
  int idx;
};
template <int NT>
__device__ __forceinline__ Extremes extremes_of(const SampleArgs& a, int row) {
  __shared__ float smx[NT / 64], smn[NT / 64];
  __shared__ int sidx[NT / 64];
  Extremes e{-INFINITY, INFINITY, 0x7FFFFFFF};
  for (int i = threadIdx.x; i < a.chunks; i += NT) {
    const int64_t at = (int64_t)row * a.chunks + i;
    const float v = a.cmax[at];
    const int id = a.cidx[at];
    if (v > e.mx || (v == e.mx && id < e.idx)) e.mx = v, e.idx = id;
    e.mn = fminf(e.mn, a.cmin[at]);
  }
#pragma unroll
  for (int o = 32; o >= 1; o >>= 1) {
    const float v = __shfl_xor(e.mx, o, 64);
    const int id = __shfl_xor(e.idx, o, 64);
    if (v > e.mx || (v == e.mx && id < e.idx)) e.mx = v, e.idx = id;
    e.mn = fminf(e.mn, __shfl_xor(e.mn, o, 64));
  }
  if ((threadIdx.x & 63) == 0) smx[threadIdx.x >> 6] = e.mx, smn[threadIdx.x >> 6] = e.mn, sidx[threadIdx.x >> 6] = e.idx;
  __syncthreads();
#pragma unroll
  for (int k = 0; k < NT / 64; ++k) {
    if (smx[k] > e.mx || (smx[k] == e.mx && sidx[k] < e.idx)) e.mx = smx[k], e.idx = sidx[k];
    e.mn = fminf(e.mn, smn[k]);
  }
  return e;
}
// Bins per neper: the row's own span, at most kSpan.
__device__ __forceinline__ double bins_of(const Extremes& e, double inv_t) {
  double span = -log_weight(e.mn, e.mx, inv_t);
  span = span < kSpan ? span : kSpan;
  return span > 0.0 ? kBins / span : 0.0;
}
__device__ __forceinline__ uint32_t bin_of(double y, double bins) { return min((uint32_t)(-y * bins), (uint32_t)kBins - 1); }

template <int TYPE>
__global__ __launch_bounds__(kT) void sample_max_kernel(SampleArgs a) {
  __shared__ float smx[kT / 64], smn[kT / 64];
  __shared__ int sidx[kT / 64];
  const int row = blockIdx.y, ch = blockIdx.x, tid = threadIdx.x;
  for (int i = ch * kT + tid; i < kBins; i += a.chunks * kT) {
    a.hmass[(int64_t)row * kBins + i] = 0;
    a.hcount[(int64_t)row * kBins + i] = 0;
  }
  if (ch == 0 && tid == 0) a.listed[row] = 0;
  bool vec;
  const void* p = row_of<TYPE>(a, row, vec);
  float mx = -INFINITY, mn = INFINITY;
  int idx = 0x7FFFFFFF;
  const int end = min(a.vocab, (ch + 1) * a.chunk);
  for (int i = ch * a.chunk + 8 * tid; i < end; i += 8 * kT) {
    float x[8];
    logits8<TYPE>(a, p, vec, i, x);
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      if (x[e] > mx) mx = x[e], idx = i + e;
      if (x[e] > -INFINITY) mn = fminf(mn, x[e]);
    }
  }
#pragma unroll
  for (int o = 32; o >= 1; o >>= 1) {
    const float v = __shfl_xor(mx, o, 64);
    const int id = __shfl_xor(idx, o, 64);
    if (v > mx || (v == mx && id < idx)) mx = v, idx = id;
    mn = fminf(mn, __shfl_xor(mn, o, 64));
  }
  if ((tid & 63) == 0) smx[tid >> 6] = mx, smn[tid >> 6] = mn, sidx[tid >> 6] = idx;
  __syncthreads();
  if (tid == 0) {
#pragma unroll
    for (int k = 1; k < kT / 64; ++k) {
      if (smx[k] > mx || (smx[k] == mx && sidx[k] < idx)) mx = smx[k], idx = sidx[k];
      mn = fminf(mn, smn[k]);
    }
    const int64_t at = (int64_t)row * a.chunks + ch;
    a.cmax[at] = mx;
    a.cmin[at] = mn;
    a.cidx[at] = idx;
  }
}

template <int TYPE>
__global__ __launch_bounds__(kT) void sample_mass_kernel(SampleArgs a) {
  __shared__ u64 hm[kBins];
  __shared__ uint32_t hc[kBins];
  __shared__ u64 red[kT / 64];
  const int row = blockIdx.y, ch = blockIdx.x, tid = threadIdx.x;
  const Setting s = setting_of(a, row);
  if (s.greedy) return;
  const bool bins_on = s.k_on || s.p_on;
  const Extremes ex = extremes_of<kT>(a, row);
  const double bins = bins_of(ex, s.inv_t);
  if (bins_on) {
    for (int i = tid; i < kBins; i += kT) hm[i] = 0, hc[i] = 0;
    __syncthreads();
  }
  bool vec;
  const void* p = row_of<TYPE>(a, row, vec);
  const int end = min(a.vocab, (ch + 1) * a.chunk);
  u64 sum = 0;
  for (int i = ch * a.chunk + 8 * tid; i < end; i += 8 * kT) {
    float x[8];
    logits8<TYPE>(a, p, vec, i, x);
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const double y = log_weight(x[e], ex.mx, s.inv_t);
      if (x[e] > -INFINITY && y >= -kSpan) {
        const double w = weight_of(y);
        if (bins_on) {
          const uint32_t b = bin_of(y, bins);
          atomicAdd(&hm[b], mass_of(w));
          atomicAdd(&hc[b], 1u);
        } else if (w >= s.min_p) {
          sum += mass_of(w);
        }
      }
    }
  }
  if (!bins_on) {
    u64 total;
    block_prefix<kT>(sum, red, total);
    if (tid == 0) a.cmass[(int64_t)row * a.chunks + ch] = total;
    return;
  }
  __syncthreads();
  for (int i = tid; i < kBins; i += kT)
    if (hc[i]) {
      atomicAdd(&a.hmass[(int64_t)row * kBins + i], hm[i]);
      atomicAdd(&a.hcount[(int64_t)row * kBins + i], hc[i]);
    }
}

// The mass that top-p asks of a kept mass M.
__device__ __forceinline__ u64 wanted(double p, u64 M) {
  const u64 t = (u64)ceil(p * (double)M);
  return t < 1 ? 1 : t > M ? M : t;
}

template <int TYPE>
__global__ __launch_bounds__(kT) void sample_list_kernel(SampleArgs a) {
  constexpr int E = kBins / kT;
  __shared__ u64 red[kT / 64];
  __shared__ uint32_t red32[kT / 64];
  __shared__ Cut cut;
  const int row = blockIdx.y, ch = blockIdx.x, tid = threadIdx.x;
  const Setting s = setting_of(a, row);
  if (!s.k_on && !s.p_on) return;          // (greedy rows have neither)
  const Extremes ex = extremes_of<kT>(a, row);
  const double bins = bins_of(ex, s.inv_t);
  // the bins of the threshold
  u64 m[E], mass = 0, all_mass;
  uint32_t c[E], count = 0, all_count;
#pragma unroll
  for (int e = 0; e < E; ++e) {
    m[e] = a.hmass[(int64_t)row * kBins + tid * E + e];
    c[e] = a.hcount[(int64_t)row * kBins + tid * E + e];
    mass += m[e];
    count += c[e];
  }
  const u64 m_before = block_prefix<kT>(mass, red, all_mass) - mass;
  const uint32_t c_before = block_prefix<kT>(count, red32, all_count) - count;
  if (tid == 0) cut = Cut{~0u, ~0u, ~0u, ~0u, 0, 0, all_mass, 0};
  __syncthreads();
  const bool k_cut = s.k_on && s.k < all_count;
  if (k_cut) {
    u64 mb = m_before;
    uint32_t cb = c_before;
#pragma unroll
    for (int e = 0; e < E; ++e) {
      if (cb < s.k && s.k <= cb + c[e]) cut.k_bin = tid * E + e, cut.before_k = cb, cut.in_k = c[e], cut.mass_k = mb;
      mb += m[e];
      cb += c[e];
    }
  }
  __syncthreads();
  if (s.p_on) {
    const u64 least = wanted(s.p, cut.mass_k);
    u64 most_mass = cut.mass_k;
    if (k_cut) most_mass += a.hmass[(int64_t)row * kBins + cut.k_bin];
    const u64 most = wanted(s.p, most_mass);
    u64 mb = m_before;
#pragma unroll
    for (int e = 0; e < E; ++e) {
      if (mb < least && least <= mb + m[e]) cut.p_first = tid * E + e, cut.mass_p = mb;
      if (mb < most && most <= mb + m[e]) cut.p_last = tid * E + e;
      mb += m[e];
    }
  }
  __syncthreads();
  if (tid == 0) {
    cut.sure = s.p_on ? cut.p_first : cut.k_bin;
    if (ch == 0) a.cut[row] = cut;
  }
  __syncthreads();
  const uint32_t sure = s.p_on ? cut.p_first : cut.k_bin;
  // their tokens, and the mass above them
  bool vec;
  const void* p = row_of<TYPE>(a, row, vec);
  const int end = min(a.vocab, (ch + 1) * a.chunk);
  u64 sum = 0;
  for (int i = ch * a.chunk + 8 * tid; i < end; i += 8 * kT) {
    float x[8];
    logits8<TYPE>(a, p, vec, i, x);
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const double y = log_weight(x[e], ex.mx, s.inv_t);
      if (!(x[e] > -INFINITY && y >= -kSpan)) continue;
      const uint32_t b = bin_of(y, bins);
      if (b < sure) {
        const double w = weight_of(y);
        if (w >= s.min_p) sum += mass_of(w);
      } else if ((b >= cut.p_first && b <= cut.p_last && s.p_on) || b == cut.k_bin) {
        const uint32_t at = atomicAdd(&a.listed[row], 1u);
        if (at < kList) a.list[(int64_t)row * kList + at] = place_of(x[e], i + e);
      }
    }
  }
  u64 total;
  block_prefix<kT>(sum, red, total);
  if (tid == 0) a.cmass[(int64_t)row * a.chunks + ch] = total;
}

__device__ __forceinline__ double weight_at(u64 place, const Extremes& ex, double inv_t) {
  const double y = log_weight(unordered((uint32_t)(place >> 32)), ex.mx, inv_t);
  return y >= -kSpan ? weight_of(y) : 0.0;
}

// Threshold of a row whose list is not whole (many tokens of one value): built
// bit by bit, a pass over the row each, first for top-k, then for top-p.
template <int TYPE>
__device__ u64 threshold_by_passes(const SampleArgs& a, const Setting& s, const Extremes& ex, const void* p, bool vec,
                                   bool k_cut, u64* red) {
  auto above = [&](u64 thr, u64& mass) {
    u64 n = 0, m = 0, total;
    for (int i = 8 * (int)threadIdx.x; i < a.vocab; i += 8 * kDrawT) {
      float x[8];
      logits8<TYPE>(a, p, vec, i, x);
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const double y = log_weight(x[e], ex.mx, s.inv_t);
        if (x[e] > -INFINITY && y >= -kSpan && place_of(x[e], i + e) >= thr) {
          ++n;
          m += mass_of(weight_of(y));
        }
      }
    }
    block_prefix<kDrawT>(m, red, mass);
    block_prefix<kDrawT>(n, red, total);
    return total;
  };
  // (bits 20 .. 31, the upper ones of an index's complement, are set in every place)
  constexpr u64 kSet = 0xFFF00000ull;
  u64 thr = kSet, M;
  if (k_cut)
    for (int bit = 63; bit >= 0; bit = bit == 32 ? 19 : bit - 1) {
      const u64 t = thr | 1ull << bit;
      if (above(t, M) >= s.k) thr = t;
    }
  if (s.p_on) {
    above(thr, M);
    const u64 want = wanted(s.p, M);
    u64 pt = kSet;
    for (int bit = 63; bit >= 0; bit = bit == 32 ? 19 : bit - 1) {
      const u64 t = pt | 1ull << bit;
      above(t, M);
      if (M >= want) pt = t;
    }
    thr = pt > thr ? pt : thr;
  }
  return thr;
}

template <int TYPE>
__global__ __launch_bounds__(kDrawT) void sample_draw_kernel(SampleArgs a) {
  __shared__ u64 place[kList];
  __shared__ u64 prefix[kList];
  __shared__ u64 cm[kMaxChunks];
  __shared__ u64 red[kDrawT / 64];
  __shared__ uint32_t first;
  __shared__ uint32_t in_chunk;
  __shared__ u64 before_chunk;
  const int row = blockIdx.x, tid = threadIdx.x;
  const Setting s = setting_of(a, row);
  const Extremes ex = extremes_of<kDrawT>(a, row);
  const int32_t step = a.state ? a.state[1] : 0;
  const int64_t u_at = a.state ? (step < 0 ? 0 : step >= a.n_u ? a.n_u - 1 : step) : row;
  __syncthreads();                         // every thread has read the state that the one that finds the token writes
  auto finish = [&](int64_t token, double logp) {
    a.token[row] = token;
    if (a.logprob) a.logprob[row] = (float)logp;
    if (a.state) {
      if (a.history && step >= 0 && step < a.history_len) a.history[step] = (int32_t)token;
      a.state[0] += 1;
      a.state[1] = step + 1;
    }
  };
  if (ex.mx == -INFINITY || s.greedy) {
    if (tid == 0) ex.mx == -INFINITY ? finish(-1, -INFINITY) : finish(ex.idx, 0.0);
    return;
  }
  bool vec;
  const void* p = row_of<TYPE>(a, row, vec);
  const bool filtered = s.k_on || s.p_on;
  u64 thr = 0;
  for (int i = tid; i < a.chunks; i += kDrawT) cm[i] = a.cmass[(int64_t)row * a.chunks + i];
  if (filtered) {
    const Cut cut = a.cut[row];
    const bool k_cut = cut.k_bin != ~0u;
    const uint32_t n = a.listed[row];
    if (n > kList) {
      thr = threshold_by_passes<TYPE>(a, s, ex, p, vec, k_cut, red);
      for (int i = tid; i < a.chunks; i += kDrawT) cm[i] = 0;
      __syncthreads();
      for (int i = 8 * tid; i < a.vocab; i += 8 * kDrawT) {
        float x[8];
        logits8<TYPE>(a, p, vec, i, x);
        u64 sum = 0;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const double y = log_weight(x[e], ex.mx, s.inv_t);
          if (x[e] > -INFINITY && y >= -kSpan && place_of(x[e], i + e) >= thr) {
            const double w = weight_of(y);
            if (w >= s.min_p) sum += mass_of(w);
          }
        }
        if (sum) atomicAdd(&cm[i / a.chunk], sum);              // (a chunk is a multiple of 8)
      }
    } else if (n) {
      // the list in descending order (bitonic), padded with zeros
      int size = 64;
      while (size < (int)n) size *= 2;
      for (int i = tid; i < size; i += kDrawT) place[i] = i < (int)n ? a.list[(int64_t)row * kList + i] : 0;
      for (int w = 2; w <= size; w *= 2)
        for (int h = w / 2; h >= 1; h /= 2) {
          __syncthreads();
          for (int i = tid; i < size / 2; i += kDrawT) {
            const int lo = 2 * i - (i & (h - 1)), hi = lo + h;
            const u64 x = place[lo], y = place[hi];
            if ((x < y) == ((lo & w) == 0)) place[lo] = y, place[hi] = x;
          }
        }
      __syncthreads();
      // inclusive masses, 4 consecutive entries per thread
      u64 m[kList / kDrawT], sum = 0, total;
#pragma unroll
      for (int e = 0; e < kList / kDrawT; ++e) {
        const int i = tid * (kList / kDrawT) + e;
        m[e] = i < (int)n ? mass_of(weight_at(place[i], ex, s.inv_t)) : 0;
        sum += m[e];
      }
      u64 before = block_prefix<kDrawT>(sum, red, total) - sum;
#pragma unroll
      for (int e = 0; e < kList / kDrawT; ++e) {
        before += m[e];
        prefix[tid * (kList / kDrawT) + e] = before;
      }
      uint32_t last = n - 1;                                    // the last entry that top-k keeps
      u64 M = cut.mass_k;
      if (tid == 0) first = n;
      __syncthreads();
      if (k_cut) {                                              // its bin's tokens are the list's last
        const uint32_t from = n - cut.in_k;
        last = from + (s.k - cut.before_k) - 1;
        M += prefix[last] - (from ? prefix[from - 1] : 0);
      }
      if (s.p_on) {
        const u64 want = wanted(s.p, M);
#pragma unroll
        for (int e = 0; e < kList / kDrawT; ++e) {
          const uint32_t i = tid * (kList / kDrawT) + e;
          if (i < n && cut.mass_p + prefix[i] >= want && (i == 0 || cut.mass_p + prefix[i - 1] < want)) first = i;
        }
        __syncthreads();
        last = min(last, first);
      }
      thr = place[last];
#pragma unroll
      for (int e = 0; e < kList / kDrawT; ++e) {
        const uint32_t i = tid * (kList / kDrawT) + e;
        if (i <= last) {
          const double w = weight_at(place[i], ex, s.inv_t);
          if (w >= s.min_p) atomicAdd(&cm[(uint32_t)~(uint32_t)place[i] / (uint32_t)a.chunk], mass_of(w));
        }
      }
    }
  }
  __syncthreads();
  // the chunk, then the token, at which the running mass passes u
  u64 total;
  const u64 mine = tid < a.chunks ? cm[tid] : 0;
  const u64 upto = block_prefix<kDrawT>(mine, red, total);
  const float uf = a.u[u_at];
  u64 want = uf > 0.f ? (u64)((double)fminf(uf, 1.f) * (double)total) : 0;
  want = want < total ? want : total - 1;
  if (upto > want && upto - mine <= want) in_chunk = tid, before_chunk = upto - mine;
  __syncthreads();
  const int c0 = (int)in_chunk * a.chunk, end = min(a.vocab, c0 + a.chunk);
  u64 passed = before_chunk;
  for (int j0 = c0; j0 < end; j0 += 8 * kDrawT) {
    const int i = j0 + 8 * tid;
    u64 m[8], sum = 0, part;
#pragma unroll
    for (int e = 0; e < 8; ++e) m[e] = 0;
    if (i < end) {
      float x[8];
      logits8<TYPE>(a, p, vec, i, x);
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const double y = log_weight(x[e], ex.mx, s.inv_t);
        if (x[e] > -INFINITY && y >= -kSpan && (!filtered || place_of(x[e], i + e) >= thr)) {
          const double w = weight_of(y);
          if (w >= s.min_p) m[e] = mass_of(w);
        }
        sum += m[e];
      }
    }
    u64 before = passed + block_prefix<kDrawT>(sum, red, part) - sum;
    if (before <= want && want < before + sum) {
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        if (before <= want && want < before + m[e]) finish(i + e, log((double)m[e] / (double)total));
        before += m[e];
      }
    }
    passed += part;
    if (passed > want) break;
  }
}

// ---------------------------------------------------------------------------
// Host side

// Chunks of 4096 logits keep a single row's steps short; from 64 rows on the
// rows fill the card and larger chunks write fewer bins.
int64_t chunk_of(int64_t rows) { return rows >= 64 ? 16384 : 4096; }

int64_t round16(int64_t n) { return (n + 15) / 16 * 16; }

struct Layout {
  int64_t cmax, cmin, cidx, cmass, hmass, hcount, listed, cut, list, bytes;
};
Layout layout_of(int64_t rows, int64_t chunks) {
  Layout l;
  int64_t at = 0;
  auto take = [&](int64_t n) {
    const int64_t here = at;
    at += round16(n);
    return here;
  };
  l.cmax = take(rows * chunks * 4);
  l.cmin = take(rows * chunks * 4);
  l.cidx = take(rows * chunks * 4);
  l.cmass = take(rows * chunks * 8);
  l.hmass = take(rows * kBins * 8);
  l.hcount = take(rows * kBins * 4);
  l.listed = take(rows * 4);
  l.cut = take(rows * (int64_t)sizeof(Cut));
  l.list = take(rows * kList * 8);
  l.bytes = at;
  return l;
}

template <int TYPE>
void launch(const SampleArgs& a, int64_t rows, bool any_draw, bool any_filter, hipStream_t st) {
  const dim3 grid((unsigned)a.chunks, (unsigned)rows);
  hipLaunchKernelGGL(sample_max_kernel<TYPE>, grid, dim3(kT), 0, st, a);
  if (any_draw) hipLaunchKernelGGL(sample_mass_kernel<TYPE>, grid, dim3(kT), 0, st, a);
  if (any_filter) hipLaunchKernelGGL(sample_list_kernel<TYPE>, grid, dim3(kT), 0, st, a);
  hipLaunchKernelGGL(sample_draw_kernel<TYPE>, dim3((unsigned)rows), dim3(kDrawT), 0, st, a);
}

}  // namespace

extern "C" int64_t bf16x_sample_workspace(int64_t rows, int64_t vocab) {
  if (rows < 0 || rows > 65535 || vocab <= 0 || vocab > kMaxVocab) return -1;
  const int64_t chunk = chunk_of(rows);
  return layout_of(rows, (vocab + chunk - 1) / chunk).bytes;
}

extern "C" int bf16x_sample(const void* logits, int32_t type, int64_t row_stride, int64_t rows, int64_t vocab,
                            const float* u, int64_t n_u, const bf16x_sample_settings* settings, int64_t* token,
                            float* logprob, int32_t* state, int32_t* history, int64_t history_len, void* workspace,
                            int64_t workspace_bytes, bf16x_stream_t stream) {
  if (!logits || !u || !settings || !token || !workspace || rows < 0 || history_len < 0 || n_u < 0) return BF16X_EARG;
  if (type != BF16X_BF16 && type != BF16X_F16 && type != BF16X_F32) return BF16X_EDTYPE;
  if (vocab <= 0 || vocab > kMaxVocab || rows > 65535) return BF16X_ESHAPE;
  if (state ? rows != 1 || n_u < 1 : n_u < rows) return BF16X_ESHAPE;
  if (history && !state) return BF16X_EARG;
  const bool wide = type == BF16X_F32;
  if ((wide ? !aligned4(logits) : !aligned2(logits)) || !aligned4(u) || !aligned8(token) || !aligned4(logprob) ||
      !aligned4(state) || !aligned4(history) || !aligned16(workspace))
    return BF16X_EARG;
  const int64_t chunk = chunk_of(rows), chunks = (vocab + chunk - 1) / chunk;
  const Layout l = layout_of(rows, chunks);
  if (workspace_bytes < l.bytes) return BF16X_ECAPACITY;
  if (rows == 0) return BF16X_OK;
  char* w = (char*)workspace;
  SampleArgs a{logits, row_stride, (int)vocab, (int)chunk, (int)chunks, u, n_u, *settings, token, logprob, state,
               history, history_len, (float*)(w + l.cmax), (float*)(w + l.cmin), (int32_t*)(w + l.cidx),
               (u64*)(w + l.cmass), (u64*)(w + l.hmass), (uint32_t*)(w + l.hcount), (uint32_t*)(w + l.listed),
               (Cut*)(w + l.cut), (u64*)(w + l.list)};
  const bf16x_sample_settings& s = *settings;
  const bool draw = s.temperature || s.temperature_all > 0.f;
  const bool filter = draw && (s.top_k || s.top_p || (s.top_k_all > 0 && s.top_k_all < vocab) || s.top_p_all < 1.f);
  const hipStream_t st = (hipStream_t)stream;
  if (wide) launch<BF16X_F32>(a, rows, draw, filter, st);
  else if (type == BF16X_F16) launch<BF16X_F16>(a, rows, draw, filter, st);
  else launch<BF16X_BF16>(a, rows, draw, filter, st);
  return launch_status();
}
