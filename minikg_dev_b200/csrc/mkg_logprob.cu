// Log probabilities of given columns in rows of logits, with each row's entropy and its largest
// alternatives, and the gradient of the logits.
//
// With c = log2(e) / tau, M the row's largest candidate and y_j = (x_j - M) c, one pass keeps
//   s = sum 2^{y_j},  t = sum 2^{y_j} y_j      (fp32, rescaled when M grows)
// from which lse = M / tau + ln s, log p_j = ln 2 (y_j - log2 s), entropy = ln 2 (log2 s - t / s).
// A larger maximum M' = M + d / c turns (s, t) into 2^-d (s, t - d s).
//
// Alternatives: every thread knows the largest element it has seen and where it first met it.  The
// topk best of those per-thread maxima (value descending, then position) name threads; an element
// outside those threads has topk better ones before it, so only their elements are read again
// (from L2) and merged exactly.  The hot loop pays one comparison per 16-byte load for that.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <algorithm>
#include <cmath>

#include "mkg_common.cuh"
#include "mkg_internal.h"

namespace mkg {
namespace {

constexpr float kLn2 = 0.693147180559945309f;
constexpr float kInf = __builtin_inff();
constexpr int kTopMax = MKG_LOGPROB_TOPK_MAX;
constexpr int kThreads = 256;
constexpr int kWarps = kThreads / kWarp;
constexpr int kUnroll = 4;           // 16-byte loads in flight per thread
constexpr int64_t kNarrow = 1024;    // rows up to this width are held by one warp
constexpr int64_t kWidthMax = int64_t(1) << 30;
constexpr unsigned kFull = 0xffffffffu;

struct Rows {
  int64_t rows, stride, mask_stride;
  int width, targets, topk;
  float c, inv_tau;  // log2(e) / tau, 1 / tau
};

struct Outputs {
  float* logprobs;
  float* entropy;
  float* lse;
  int64_t* top_ids;
  float* top_logprobs;
  float* stats;
  unsigned* err;
};

template <typename T> __device__ __forceinline__ float to_f32(T v);
template <> __device__ __forceinline__ float to_f32(float v) { return v; }
template <> __device__ __forceinline__ float to_f32(__nv_bfloat16 v) { return __bfloat162float(v); }
template <> __device__ __forceinline__ float to_f32(__half v) { return __half2float(v); }
template <typename T> __device__ __forceinline__ T from_f32(float v);
template <> __device__ __forceinline__ float from_f32(float v) { return v; }
template <> __device__ __forceinline__ __nv_bfloat16 from_f32(float v) { return __float2bfloat16_rn(v); }
template <> __device__ __forceinline__ __half from_f32(float v) { return __float2half_rn(v); }

// 2^y, relative error about 2^-22; results below 2^-126 are 0
__device__ __forceinline__ float ex2(float y) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(y));
  return r;
}
// max that keeps a NaN (fmaxf drops it)
__device__ __forceinline__ float max_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}
// y = (x - m) c with -inf brought to where 2^y is 0 but y stays finite (0 * y must be 0)
__device__ __forceinline__ float scaled(float x, float m, float c) { return max_nan((x - m) * c, -256.0f); }

template <typename T> constexpr int kVec = 16 / sizeof(T);

// A row cut into 16-byte slots: slot q holds the columns [q * kVec - lead, + kVec) of the row, so
// that whole slots start on 16-byte addresses whatever the row's own alignment is.
template <typename T> struct RowView {
  const T* x;
  const uint8_t* mask;
  int width, lead, slots;
  bool mask_vec;  // whole slots of the mask are aligned too

  __device__ __forceinline__ RowView(const T* x_, const uint8_t* mask_, int width_) : x(x_), mask(mask_), width(width_) {
    lead = static_cast<int>((reinterpret_cast<uintptr_t>(x) / sizeof(T)) % kVec<T>);
    slots = (width + lead + kVec<T> - 1) / kVec<T>;
    mask_vec = mask == nullptr || (reinterpret_cast<uintptr_t>(mask) - lead) % kVec<T> == 0;
  }
  __device__ __forceinline__ int first(int slot) const { return slot * kVec<T> - lead; }

  // the slot's logits in fp32; columns outside the row and non-candidates as -inf
  template <bool kMask> __device__ __forceinline__ void load(int slot, float (&v)[kVec<T>]) const {
    const int j0 = first(slot);
    if (j0 >= 0 && j0 + kVec<T> <= width) {
      const uint4 raw = __ldg(reinterpret_cast<const uint4*>(x + j0));
      T e[kVec<T>];
      memcpy(e, &raw, 16);
#pragma unroll
      for (int i = 0; i < kVec<T>; ++i) v[i] = to_f32<T>(e[i]);
      if (kMask) {
        uint8_t on[kVec<T>];
        if (mask_vec) {
          if constexpr (kVec<T> == 4) {
            const uint32_t b = __ldg(reinterpret_cast<const uint32_t*>(mask + j0));
            memcpy(on, &b, 4);
          } else {
            const uint2 b = __ldg(reinterpret_cast<const uint2*>(mask + j0));
            memcpy(on, &b, 8);
          }
        } else {
#pragma unroll
          for (int i = 0; i < kVec<T>; ++i) on[i] = __ldg(mask + j0 + i);
        }
#pragma unroll
        for (int i = 0; i < kVec<T>; ++i)
          if (!on[i]) v[i] = -kInf;
      }
    } else {
#pragma unroll
      for (int i = 0; i < kVec<T>; ++i) {
        const int j = j0 + i;
        const bool in = j >= 0 && j < width && (!kMask || __ldg(mask + j) != 0);
        v[i] = in ? to_f32<T>(x[j]) : -kInf;
      }
    }
  }
};

// (value, column) as one word: larger values first, on equal values the lower column; 0 = none
__device__ __forceinline__ unsigned long long rank_key(float v, uint32_t at) { return pack_value_rank(v + 0.0f, at); }

__device__ __forceinline__ unsigned long long shfl_xor64(unsigned long long v, int o) {
  return __shfl_xor_sync(kFull, v, o);
}

// One step of a bitonic network over the warp: keep the larger of the pair (lane, lane ^ o) if `up`.
__device__ __forceinline__ unsigned long long exchange(unsigned long long v, int o, bool up) {
  const unsigned long long w = shfl_xor64(v, o);
  return (w > v) == up ? w : v;
}
// The 32 keys of a warp in ascending order of the lanes.
__device__ __forceinline__ unsigned long long sort_ascending(unsigned long long v, int lane) {
#pragma unroll
  for (int size = 2; size <= 32; size <<= 1)
#pragma unroll
    for (int o = size >> 1; o > 0; o >>= 1) v = exchange(v, o, ((lane & o) != 0) == ((lane & size) == 0 || size == 32));
  return v;
}
// `best` descending over the lanes, `add` ascending: the 32 largest of both, descending.
__device__ __forceinline__ unsigned long long merge_best(unsigned long long best, unsigned long long add, int lane) {
  unsigned long long v = best > add ? best : add;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v = exchange(v, o, (lane & o) == 0);
  return v;
}

struct Moments {
  float m, s, t;  // largest, sum 2^y, sum 2^y y
};
// (m, s, t) seen from a larger maximum M.  Without a candidate m is -inf and s is 0, or NaN where
// the values were NaN: it passes as it is.
__device__ __forceinline__ void shift_to(Moments& a, float M, float c) {
  if (a.m == M || a.m == -kInf) return;
  const float d = (a.m - M) * c;
  const float f = ex2(d);
  a.t = f * fmaf(d, a.s, a.t);
  if (f == 0.0f) a.t = a.s - a.s;  // far below: no share, 0 * d would not be 0 for an infinite d
  a.s = f * a.s;
}
__device__ __forceinline__ Moments warp_join(Moments a, float c) {
  float M = a.m;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) M = fmaxf(M, __shfl_xor_sync(kFull, M, o));
  shift_to(a, M, c);
  return {M, warp_sum(a.s), warp_sum(a.t)};
}

// The outputs of one row by the threads of a warp or block (`first` of `count`); `best`: the row's
// largest keys, descending over the lanes of the threads with lane < 32 of the first warp.
template <typename T>
__device__ __forceinline__ void finish_row(const Rows& r, const Outputs& o, int64_t row, const T* x,
                                           const uint8_t* mask, const int64_t* targets, Moments a,
                                           unsigned long long best, int first, int count) {
  const bool none = a.m == -kInf && a.s == 0.0f;
  const float log2s = none ? -kInf : a.s == a.s ? log2f(a.s) : a.s;
  if (first == 0) {
    o.lse[row] = none ? -kInf : fmaf(log2s, kLn2, a.m * r.inv_tau) + (a.s - a.s);
    o.entropy[row] = none ? 0.0f : fmaxf(kLn2 * (log2s - a.t / a.s), 0.0f) + (a.s - a.s);
    o.stats[2 * row] = a.m;
    o.stats[2 * row + 1] = log2s;
  }
  for (int q = first; q < r.targets; q += count) {
    const int64_t t = targets[row * r.targets + q];
    float lp = 0.0f;
    if (t < -1 || t >= r.width) {
      raise_flag(o.err, MKG_DEV_BAD_TARGET);
      lp = __int_as_float(0x7fc00000);
    } else if (t >= 0) {
      const bool on = mask == nullptr || mask[t] != 0;
      if (none) lp = -kInf;
      else if (!on) lp = -kInf + (a.s - a.s);
      else lp = kLn2 * ((to_f32<T>(x[t]) - a.m) * r.c - log2s);
    }
    o.logprobs[row * r.targets + q] = lp;
  }
  if (first < r.topk) {
    const bool nan = !(a.s == a.s);
    const bool have = best != 0 && !nan;
    o.top_ids[row * r.topk + first] = have ? static_cast<int64_t>(packed_rank(best)) : -1;
    o.top_logprobs[row * r.topk + first] =
        nan ? a.s : have ? kLn2 * ((packed_value(best) - a.m) * r.c - log2s) : -kInf;
  }
}

// ---------------------------------------------------------------- rows of up to 1024 columns: a warp each
template <typename T, bool kMask, int kPer>
__global__ void __launch_bounds__(kThreads) logprob_narrow_kernel(Rows r, const T* __restrict__ logits,
                                                                  const uint8_t* __restrict__ masks,
                                                                  const int64_t* __restrict__ targets, Outputs o) {
  const int lane = threadIdx.x & 31;
  const int64_t row = static_cast<int64_t>(blockIdx.x) * kWarps + (threadIdx.x >> 5);
  if (row >= r.rows) return;
  const T* x = logits + row * r.stride;
  const uint8_t* mask = kMask ? masks + row * r.mask_stride : nullptr;
  float v[kPer];
  Moments a{-kInf, 0.0f, 0.0f};
#pragma unroll
  for (int i = 0; i < kPer; ++i) {
    const int j = i * kWarp + lane;
    v[i] = j < r.width && (!kMask || mask[j] != 0) ? to_f32<T>(x[j]) : -kInf;
    a.m = fmaxf(a.m, v[i]);
  }
#pragma unroll
  for (int off = 16; off > 0; off >>= 1) a.m = fmaxf(a.m, __shfl_xor_sync(kFull, a.m, off));
  const float from = a.m == -kInf ? 0.0f : a.m;
#pragma unroll
  for (int i = 0; i < kPer; ++i) {
    const float y = scaled(v[i], from, r.c);
    const float e = ex2(y);
    a.s += e;
    a.t = fmaf(e, y, a.t);
  }
  a.s = warp_sum(a.s);
  a.t = warp_sum(a.t);
  unsigned long long best = 0;
  if (r.topk > 0) {
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
      unsigned long long k = v[i] > -kInf ? rank_key(v[i], i * kWarp + lane) : 0;
      const unsigned long long worst = __shfl_sync(kFull, best, r.topk - 1);
      if (__any_sync(kFull, k > worst)) best = merge_best(best, sort_ascending(k, lane), lane);
    }
  }
  finish_row<T>(r, o, row, x, mask, targets, a, best, lane, kWarp);
}

// ---------------------------------------------------------------- wider rows: blocks, joined if several
struct Partial {
  float m, s, t, pad;
};

template <typename T, bool kMask, bool kTop>
__global__ void __launch_bounds__(kThreads) logprob_wide_kernel(Rows r, const T* __restrict__ logits,
                                                                const uint8_t* __restrict__ masks,
                                                                const int64_t* __restrict__ targets, Outputs o,
                                                                int splits, int slots_per_split,
                                                                Partial* __restrict__ partials,
                                                                unsigned long long* __restrict__ keys) {
  __shared__ float sh_m[kWarps], sh_s[kWarps], sh_t[kWarps];
  __shared__ unsigned long long sh_key[kThreads];
  __shared__ int sh_winner[kWarp];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int64_t row = blockIdx.x / splits;
  const int split = static_cast<int>(blockIdx.x % splits);
  const T* x = logits + row * r.stride;
  const uint8_t* mask = kMask ? masks + row * r.mask_stride : nullptr;
  const RowView<T> view(x, mask, r.width);
  const int lo = split * slots_per_split;
  const int hi = min(lo + slots_per_split, view.slots);

  Moments a{-kInf, 0.0f, 0.0f};
  int at = 0;  // the slot where the thread first met a.m
  for (int base = lo + tid; base < hi; base += kThreads * kUnroll) {
    float v[kUnroll][kVec<T>];
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) {
      const int slot = base + u * kThreads;
      if (slot < hi) {
        view.template load<kMask>(slot, v[u]);
      } else {
#pragma unroll
        for (int i = 0; i < kVec<T>; ++i) v[u][i] = -kInf;
      }
    }
    float M = a.m;
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) {
      float big = v[u][0];
#pragma unroll
      for (int i = 1; i < kVec<T>; ++i) big = fmaxf(big, v[u][i]);
      if (big > M) {
        M = big;
        at = base + u * kThreads;
      }
    }
    if (M > a.m) {
      shift_to(a, M, r.c);
      a.m = M;
    }
    const float from = M == -kInf ? 0.0f : M;
#pragma unroll
    for (int u = 0; u < kUnroll; ++u)
#pragma unroll
      for (int i = 0; i < kVec<T>; ++i) {
        const float y = scaled(v[u][i], from, r.c);
        const float e = ex2(y);
        a.s += e;
        a.t = fmaf(e, y, a.t);
      }
  }
  const unsigned long long mine = a.m > -kInf ? rank_key(a.m, static_cast<uint32_t>(at)) : 0;

  Moments all = warp_join(a, r.c);
  if (lane == 0) {
    sh_m[warp] = all.m;
    sh_s[warp] = all.s;
    sh_t[warp] = all.t;
  }
  unsigned long long best = 0;
  if (kTop) sh_key[tid] = sort_ascending(mine, lane);
  __syncthreads();
  {
    Moments b = lane < kWarps ? Moments{sh_m[lane], sh_s[lane], sh_t[lane]} : Moments{-kInf, 0.0f, 0.0f};
    all = warp_join(b, r.c);
  }
  if (kTop) {
    // the topk best threads, by (largest element, where it was first met)
    unsigned long long top = 0;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) top = merge_best(top, sh_key[w * kWarp + lane], lane);
    // a slot's position names its thread: slots are dealt out in turn
    if (warp == 0)
      sh_winner[lane] = top != 0 && lane < r.topk
                            ? static_cast<int>((packed_rank(top) - static_cast<uint32_t>(lo)) % kThreads) : -1;
    const unsigned long long floor_key = __shfl_sync(kFull, top, r.topk - 1);
    const float least = floor_key != 0 ? packed_value(floor_key) : -kInf;
    const uint32_t least_slot = floor_key != 0 ? packed_rank(floor_key) : 0xffffffffu;
    __syncthreads();
    for (int w = warp; w < r.topk; w += kWarps) {
      const int who = sh_winner[w];
      if (who < 0) continue;
      for (int base = lo + who; base < hi; base += kThreads * kWarp) {
        const int slot = base + lane * kThreads;
        float v[kVec<T>];
        if (slot < hi) {
          view.template load<kMask>(slot, v);
        } else {
#pragma unroll
          for (int i = 0; i < kVec<T>; ++i) v[i] = -kInf;
        }
#pragma unroll
        for (int i = 0; i < kVec<T>; ++i) {
          const bool in = v[i] > least || (v[i] == least && v[i] > -kInf && static_cast<uint32_t>(slot) <= least_slot);
          const unsigned long long k = in ? rank_key(v[i], static_cast<uint32_t>(view.first(slot) + i)) : 0;
          const unsigned long long worst = __shfl_sync(kFull, best, r.topk - 1);
          if (__any_sync(kFull, k > worst)) best = merge_best(best, sort_ascending(k, lane), lane);
        }
      }
    }
    __syncthreads();
    sh_key[warp * kWarp + (31 - lane)] = best;  // ascending
    __syncthreads();
    best = 0;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) best = merge_best(best, sh_key[w * kWarp + lane], lane);
  }
  if (splits == 1) {
    finish_row<T>(r, o, row, x, mask, targets, all, best, tid, kThreads);
  } else {
    const int64_t at_split = row * splits + split;
    if (tid == 0) partials[at_split] = {all.m, all.s, all.t, 0.0f};
    if (kTop && tid < r.topk) keys[at_split * r.topk + tid] = best;
  }
}

// One block per row joins its splits in their order.
template <typename T, bool kMask>
__global__ void __launch_bounds__(kThreads) logprob_join_kernel(Rows r, const T* __restrict__ logits,
                                                                const uint8_t* __restrict__ masks,
                                                                const int64_t* __restrict__ targets, Outputs o,
                                                                int splits, const Partial* __restrict__ partials,
                                                                const unsigned long long* __restrict__ keys) {
  __shared__ float sh_m[kWarps], sh_s[kWarps], sh_t[kWarps];
  __shared__ unsigned long long sh_key[kThreads];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int64_t row = blockIdx.x;
  Moments a{-kInf, 0.0f, 0.0f};
  for (int i = tid; i < splits; i += kThreads) {
    const Partial p = partials[row * splits + i];
    Moments b{p.m, p.s, p.t};
    const float M = fmaxf(a.m, b.m);
    shift_to(a, M, r.c);
    shift_to(b, M, r.c);
    a = {M, a.s + b.s, a.t + b.t};
  }
  Moments all = warp_join(a, r.c);
  if (lane == 0) {
    sh_m[warp] = all.m;
    sh_s[warp] = all.s;
    sh_t[warp] = all.t;
  }
  unsigned long long best = 0;
  const int n = splits * r.topk;  // 0: nothing to merge
  for (int i = warp * kWarp; i < n; i += kThreads) {
    const unsigned long long k = i + lane < n ? keys[row * n + i + lane] : 0;
    const unsigned long long worst = __shfl_sync(kFull, best, r.topk - 1);
    if (__any_sync(kFull, k > worst)) best = merge_best(best, sort_ascending(k, lane), lane);
  }
  sh_key[warp * kWarp + (31 - lane)] = best;
  __syncthreads();
  Moments b = lane < kWarps ? Moments{sh_m[lane], sh_s[lane], sh_t[lane]} : Moments{-kInf, 0.0f, 0.0f};
  all = warp_join(b, r.c);
  best = 0;
#pragma unroll
  for (int w = 0; w < kWarps; ++w) best = merge_best(best, sh_key[w * kWarp + lane], lane);
  const T* x = logits + row * r.stride;
  finish_row<T>(r, o, row, x, kMask ? masks + row * r.mask_stride : nullptr, targets, all, best, tid, kThreads);
}

// ---------------------------------------------------------------- gradient
struct Upstream {
  const int64_t* targets;
  const int64_t* top_ids;
  const float* entropy;
  const float* stats;
  const float* logprobs;  // gradients of the outputs, each may be null
  const float* g_entropy;
  const float* lse;
  const float* top;
};

// dx_j = p_j (a + b log2 p_j) for candidates, with p_j = 2^{log2 p_j}, plus the named columns' own
// gradients / tau.
struct RowGrad {
  float m, log2s, a, b;
  bool none;
};

// The gradient that arrives at named column q of the row (targets first, then alternatives) and
// which column that is; -1: none.
__device__ __forceinline__ float named(const Rows& r, const Upstream& u, int64_t row, int q, int64_t& id) {
  float g = 0.0f;
  if (q < r.targets) {
    id = u.logprobs ? u.targets[row * r.targets + q] : -1;
    if (id >= 0 && id < r.width) g = u.logprobs[row * r.targets + q];
  } else {
    id = u.top ? u.top_ids[row * r.topk + q - r.targets] : -1;
    if (id >= 0) g = u.top[row * r.topk + q - r.targets];
  }
  if (id < 0 || id >= r.width) id = -1;
  return g;
}

__device__ __forceinline__ RowGrad row_grad(const Rows& r, const Upstream& u, int64_t row, float named_sum) {
  RowGrad g;
  g.m = u.stats[2 * row];
  g.log2s = u.stats[2 * row + 1];
  const float gh = u.g_entropy ? u.g_entropy[row] : 0.0f;
  const float gl = u.lse ? u.lse[row] : 0.0f;
  g.a = -(named_sum + gh * u.entropy[row] - gl) * r.inv_tau;
  g.b = -gh * kLn2 * r.inv_tau;
  g.none = g.log2s == -kInf;
  return g;
}

__device__ __forceinline__ float share(const RowGrad& g, float x, float c) {
  const float y = max_nan((x - g.m) * c - g.log2s, -256.0f);
  return ex2(y) * fmaf(g.b, y, g.a);
}

template <typename T, bool kMask>
__global__ void __launch_bounds__(kThreads) logprob_backward_kernel(Rows r, const T* __restrict__ logits,
                                                                    const uint8_t* __restrict__ masks, Upstream u,
                                                                    T* __restrict__ grads, int splits,
                                                                    int slots_per_split) {
  extern __shared__ int sh_id[];  // [named], then their gradients
  __shared__ float sh_sum[kWarps];
  const int named_n = r.targets + r.topk;
  float* sh_g = reinterpret_cast<float*>(sh_id + named_n);
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int64_t row = blockIdx.x / splits;
  const int split = static_cast<int>(blockIdx.x % splits);
  const T* x = logits + row * r.stride;
  const uint8_t* mask = kMask ? masks + row * r.mask_stride : nullptr;
  T* grad = grads + row * r.width;
  const RowView<T> view(x, mask, r.width);

  float sum = 0.0f;
  for (int q = tid; q < named_n; q += kThreads) {
    int64_t id;
    const float g = named(r, u, row, q, id);
    sh_id[q] = static_cast<int>(id);
    sh_g[q] = g;
    sum += g;
  }
  sum = warp_sum(sum);
  if (lane == 0) sh_sum[warp] = sum;
  __syncthreads();
  sum = 0.0f;
#pragma unroll
  for (int w = 0; w < kWarps; ++w) sum += sh_sum[w];
  const RowGrad g = row_grad(r, u, row, sum);

  const int lo = split * slots_per_split;
  const int hi = min(lo + slots_per_split, view.slots);
  const bool store_vec = (reinterpret_cast<uintptr_t>(grad) - view.lead * sizeof(T)) % 16 == 0;
  for (int slot = lo + tid; slot < hi; slot += kThreads) {
    float v[kVec<T>];
    view.template load<kMask>(slot, v);
    const int j0 = view.first(slot);
    T out[kVec<T>];
#pragma unroll
    for (int i = 0; i < kVec<T>; ++i) {
      // a non-candidate reads as -inf: its share is 0 unless the row itself is NaN
      const bool off = g.none || (kMask && v[i] == -kInf);
      out[i] = from_f32<T>(off ? 0.0f : share(g, v[i], r.c));
    }
    if (store_vec && j0 >= 0 && j0 + kVec<T> <= r.width) {
      uint4 raw;
      memcpy(&raw, out, 16);
      *reinterpret_cast<uint4*>(grad + j0) = raw;
    } else {
#pragma unroll
      for (int i = 0; i < kVec<T>; ++i)
        if (j0 + i >= 0 && j0 + i < r.width) grad[j0 + i] = out[i];
    }
  }
  if (named_n == 0 || g.none) return;
  __syncthreads();
  // the named columns of this block again, with their own gradients added before the one rounding
  const int j_lo = view.first(lo), j_hi = view.first(hi);
  for (int q = tid; q < named_n; q += kThreads) {
    const int id = sh_id[q];
    if (id < 0 || id < j_lo || id >= j_hi || (kMask && mask[id] == 0)) continue;
    float add = 0.0f;
    bool again = false;
    for (int k = 0; k < named_n; ++k)
      if (sh_id[k] == id) {
        again |= k < q;  // the first to name the column writes it
        add += sh_g[k];
      }
    if (!again) grad[id] = from_f32<T>(fmaf(add, r.inv_tau, share(g, to_f32<T>(x[id]), r.c)));
  }
}

int check_params(const mkg_logprob_params* p, Rows* r) {
  MKG_REQUIRE(p, "logprob: null parameters");
  MKG_REQUIRE(p->rows >= 0 && p->width >= 1 && p->width <= kWidthMax, "logprob: width %lld outside [1, 2^30]",
              (long long)p->width);
  MKG_REQUIRE(p->rows <= (int64_t(1) << 30), "logprob: %lld rows, at most 2^30", (long long)p->rows);
  MKG_REQUIRE(p->targets >= 0 && p->targets <= MKG_LOGPROB_TARGETS_MAX, "logprob: %lld targets per row, at most %d",
              (long long)p->targets, (int)MKG_LOGPROB_TARGETS_MAX);
  MKG_REQUIRE(p->topk >= 0 && p->topk <= kTopMax, "logprob: topk %lld outside [0, %d]", (long long)p->topk, kTopMax);
  MKG_REQUIRE(p->dtype >= MKG_F32 && p->dtype <= MKG_F16, "logprob: unknown element type %d", p->dtype);
  MKG_REQUIRE(p->tau > 0.0 && std::isfinite(p->tau), "logprob: tau must be positive and finite");
  MKG_REQUIRE(p->row_stride >= 0 && p->mask_row_stride >= 0, "logprob: negative row stride");
  *r = Rows{p->rows, p->row_stride, p->mask_row_stride, (int)p->width, (int)p->targets, (int)p->topk,
            (float)(1.4426950408889634 / p->tau), (float)(1.0 / p->tau)};
  return MKG_OK;
}

struct Cut {
  int splits, slots;
};
// Blocks per row: enough that all rows together fill the SMs several times over, each with at
// least `least` rounds of loads.
Cut cut_rows(const mkg_logprob_params* p, int per_sm, int least) {
  const int vec = p->dtype == MKG_F32 ? 4 : 8;
  const int64_t slots = (p->width + 2 * vec - 2) / vec;  // the most a row can have
  const int64_t round = (int64_t)kThreads * kUnroll;
  const int64_t want = ((int64_t)persistent_blocks(per_sm) + p->rows - 1) / std::max<int64_t>(p->rows, 1);
  const int64_t most = std::max<int64_t>(1, slots / (round * least));
  const int64_t splits = std::max<int64_t>(1, std::min(want, most));
  int64_t per = (slots + splits - 1) / splits;
  per = (per + round - 1) / round * round;
  return {(int)((slots + per - 1) / per), (int)per};
}
Cut forward_cut(const mkg_logprob_params* p) { return cut_rows(p, 8, 1); }
Cut backward_cut(const mkg_logprob_params* p) { return cut_rows(p, 8, 1); }

template <typename F> int by_type(int32_t dtype, bool mask, F f) {
  switch (dtype) {
    case MKG_F32: return mask ? f((float*)nullptr, std::true_type()) : f((float*)nullptr, std::false_type());
    case MKG_BF16:
      return mask ? f((__nv_bfloat16*)nullptr, std::true_type()) : f((__nv_bfloat16*)nullptr, std::false_type());
    default: return mask ? f((__half*)nullptr, std::true_type()) : f((__half*)nullptr, std::false_type());
  }
}

template <typename T, bool kMask>
int launch_narrow(const Rows& r, const void* logits, const uint8_t* mask, const int64_t* targets, const Outputs& o,
                  cudaStream_t st) {
  const unsigned grid = (unsigned)((r.rows + kWarps - 1) / kWarps);
  const T* x = static_cast<const T*>(logits);
  const int per = (r.width + kWarp - 1) / kWarp;
  if (per <= 1) logprob_narrow_kernel<T, kMask, 1><<<grid, kThreads, 0, st>>>(r, x, mask, targets, o);
  else if (per <= 2) logprob_narrow_kernel<T, kMask, 2><<<grid, kThreads, 0, st>>>(r, x, mask, targets, o);
  else if (per <= 4) logprob_narrow_kernel<T, kMask, 4><<<grid, kThreads, 0, st>>>(r, x, mask, targets, o);
  else if (per <= 8) logprob_narrow_kernel<T, kMask, 8><<<grid, kThreads, 0, st>>>(r, x, mask, targets, o);
  else if (per <= 16) logprob_narrow_kernel<T, kMask, 16><<<grid, kThreads, 0, st>>>(r, x, mask, targets, o);
  else logprob_narrow_kernel<T, kMask, 32><<<grid, kThreads, 0, st>>>(r, x, mask, targets, o);
  MKG_LAUNCHED("logprob_narrow_kernel");
  return MKG_OK;
}

}  // namespace

size_t logprob_workspace_bytes(const mkg_logprob_params* p) {
  Rows r;
  if (check_params(p, &r) != MKG_OK || p->width <= kNarrow) return 0;
  const Cut cut = forward_cut(p);
  if (cut.splits == 1) return 0;
  return (size_t)(p->rows * cut.splits) * (sizeof(Partial) + (size_t)p->topk * sizeof(unsigned long long));
}

int logprob_forward(const mkg_logprob_params* p, const void* logits, const uint8_t* mask, const int64_t* targets,
                    float* logprobs, float* entropy, float* lse, int64_t* top_ids, float* top_logprobs, float* stats,
                    void* ws, size_t ws_bytes, unsigned* err, cudaStream_t st) {
  Rows r;
  if (int rc = check_params(p, &r)) return rc;
  if (p->rows == 0) return MKG_OK;
  MKG_REQUIRE(logits && entropy && lse && stats && (p->targets == 0 || (targets && logprobs)) &&
                  (p->topk == 0 || (top_ids && top_logprobs)), "logprob_forward: null argument");
  const size_t need = logprob_workspace_bytes(p);
  if (ws_bytes < need || (need > 0 && !ws)) {
    set_error("logprob_forward: workspace %zu < %zu bytes", ws_bytes, need);
    return MKG_ERR_CAPACITY;
  }
  const Outputs o{logprobs, entropy, lse, top_ids, top_logprobs, stats, err};
  return by_type(p->dtype, mask != nullptr, [&](auto* tag, auto has_mask) -> int {
    using T = std::remove_pointer_t<decltype(tag)>;
    constexpr bool kMask = decltype(has_mask)::value;
    const T* x = static_cast<const T*>(logits);
    MKG_REQUIRE(reinterpret_cast<uintptr_t>(x) % sizeof(T) == 0, "logprob_forward: misaligned logits");
    if (p->width <= kNarrow) return launch_narrow<T, kMask>(r, logits, mask, targets, o, st);
    const Cut cut = forward_cut(p);
    MKG_REQUIRE(r.rows * cut.splits < (int64_t(1) << 31), "logprob_forward: too many rows");
    Partial* partials = static_cast<Partial*>(ws);
    unsigned long long* keys = reinterpret_cast<unsigned long long*>(partials + (cut.splits > 1 ? r.rows * cut.splits : 0));
    const unsigned grid = (unsigned)(r.rows * cut.splits);
    if (r.topk > 0)
      logprob_wide_kernel<T, kMask, true><<<grid, kThreads, 0, st>>>(r, x, mask, targets, o, cut.splits, cut.slots,
                                                                     partials, keys);
    else
      logprob_wide_kernel<T, kMask, false><<<grid, kThreads, 0, st>>>(r, x, mask, targets, o, cut.splits, cut.slots,
                                                                      partials, keys);
    MKG_LAUNCHED("logprob_wide_kernel");
    if (cut.splits > 1) {
      logprob_join_kernel<T, kMask><<<(unsigned)r.rows, kThreads, 0, st>>>(r, x, mask, targets, o, cut.splits,
                                                                           partials, keys);
      MKG_LAUNCHED("logprob_join_kernel");
    }
    return MKG_OK;
  });
}

int logprob_backward(const mkg_logprob_params* p, const void* logits, const uint8_t* mask, const int64_t* targets,
                     const int64_t* top_ids, const float* entropy, const float* stats, const float* g_logprobs,
                     const float* g_entropy, const float* g_lse, const float* g_top, void* grad, cudaStream_t st) {
  Rows r;
  if (int rc = check_params(p, &r)) return rc;
  if (p->rows == 0) return MKG_OK;
  MKG_REQUIRE(logits && entropy && stats && grad && (p->targets == 0 || targets) && (p->topk == 0 || top_ids),
              "logprob_backward: null argument");
  const Upstream u{targets, top_ids, entropy, stats, g_logprobs, g_entropy, g_lse, g_top};
  return by_type(p->dtype, mask != nullptr, [&](auto* tag, auto has_mask) -> int {
    using T = std::remove_pointer_t<decltype(tag)>;
    constexpr bool kMask = decltype(has_mask)::value;
    const T* x = static_cast<const T*>(logits);
    MKG_REQUIRE(reinterpret_cast<uintptr_t>(x) % sizeof(T) == 0 && reinterpret_cast<uintptr_t>(grad) % sizeof(T) == 0,
                "logprob_backward: misaligned tensors");
    const Cut cut = backward_cut(p);
    MKG_REQUIRE(r.rows * cut.splits < (int64_t(1) << 31), "logprob_backward: too many rows");
    const size_t sh = (size_t)(r.targets + r.topk) * 8;
    logprob_backward_kernel<T, kMask><<<(unsigned)(r.rows * cut.splits), kThreads, sh, st>>>(
        r, x, mask, u, static_cast<T*>(grad), cut.splits, cut.slots);
    MKG_LAUNCHED("logprob_backward_kernel");
    return MKG_OK;
  });
}

}  // namespace mkg
