// One AdamW step over many tensors in one launch, with the moments held in 32 or in 8 bits.
//
//   m = b1 m + (1 - b1) g,   v = b2 v + (1 - b2) g^2
//   p = p (1 - lr wd) - lr / (1 - b1^t) * m / (sqrt(v) / sqrt(1 - b2^t) + eps)
//
// The tensors' addresses travel as kernel parameters, so a step copies nothing to the device and can
// be captured; the step counts live on the device and the last block to finish advances them.
//
// Moments in 8 bits.  Blocks of 256 values of a tensor share a power of two.  First moments: sign,
// 4 exponent bits, 3 of mantissa (largest 448).  Second moments are never negative, so the sign's
// bit goes to the exponent: 5 and 3 bits (largest 1.75, smallest 2^-33), a relative error of 2^-4 at
// most on v, 2^-5 on its root, over 34 binades.  A second moment above 0 is never held as 0, so that
// no update is divided by eps alone.  A power of two as scale makes scaling exact and loses nothing,
// because the held values have the same relative spacing everywhere.  The sums are taken in fp64 and
// rounded once to what is held: rounding them to fp32 first would move about one in 10^6 of them to
// the neighbouring value, and with 16-bit gradients sums on the middle of two values are frequent.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_fp8.h>

#include <algorithm>
#include <cfloat>
#include <cmath>

#include "mkg_common.cuh"
#include "mkg_internal.h"

namespace mkg {
namespace {

constexpr int kThreads = 256;
constexpr int kBlock = MKG_ADAMW_BLOCK;      // values that share a scale: a warp's share of a chunk
constexpr int kQuad = 4;                     // values per access
constexpr int kQuads = kBlock / kQuad / kWarp;  // accesses per thread
constexpr int kChunk = kThreads / kWarp * kBlock;
constexpr unsigned kFull = 0xffffffffu;
constexpr int kFirstLow = -120, kSecondLow = -90, kHigh = 120;  // exponents of the blocks' scales

// Tensors of one launch.  A launch's parameters may take 32,764 bytes.
template <int kCap> struct Table {
  void* param[kCap];
  const void* grad[kCap];
  int64_t numel[kCap];
  int32_t block[kCap];      // first block of 256 of its moments
  int32_t index[kCap];      // its step count
  int32_t chunk[kCap + 1];  // first chunk
  int32_t n;
};

struct Hyper {
  double lr, beta1, beta2, weight_decay;
  float eps;
  const float* lr_device;
};

struct State {
  void* first;
  void* second;
  float* first_scale;
  float* second_scale;
  int64_t* steps;
  unsigned* ticket;
};

// What a step's numbers come to for one tensor.
struct Rates {
  float decay, step, root;  // 1 - lr wd, lr / (1 - b1^t), 1 / sqrt(1 - b2^t)
};

template <typename T> struct Quad { T v[kQuad]; };
template <typename T> __device__ __forceinline__ float to_f32(T v);
template <> __device__ __forceinline__ float to_f32(float v) { return v; }
template <> __device__ __forceinline__ float to_f32(__nv_bfloat16 v) { return __bfloat162float(v); }
template <> __device__ __forceinline__ float to_f32(__half v) { return __half2float(v); }
template <typename T> __device__ __forceinline__ T from_f32(float v);
template <> __device__ __forceinline__ float from_f32(float v) { return v; }
template <> __device__ __forceinline__ __nv_bfloat16 from_f32(float v) { return __float2bfloat16_rn(v); }
template <> __device__ __forceinline__ __half from_f32(float v) { return __float2half_rn(v); }

template <typename T> struct Bits;
template <> struct Bits<float> { using type = uint4; };
template <> struct Bits<__nv_bfloat16> { using type = uint2; };
template <> struct Bits<__half> { using type = uint2; };

// Four values from `at`; those from `left` on read as 0.
template <typename T> __device__ __forceinline__ void load_quad(const T* at, int64_t left, bool whole, float (&out)[kQuad]) {
  if (whole && left >= kQuad) {
    using B = typename Bits<T>::type;
    const B raw = *reinterpret_cast<const B*>(at);
    T e[kQuad];
    memcpy(e, &raw, sizeof(raw));
#pragma unroll
    for (int i = 0; i < kQuad; ++i) out[i] = to_f32<T>(e[i]);
  } else {
#pragma unroll
    for (int i = 0; i < kQuad; ++i) out[i] = i < left ? to_f32<T>(at[i]) : 0.0f;
  }
}
template <typename T> __device__ __forceinline__ void store_quad(T* at, int64_t left, bool whole, const float (&v)[kQuad]) {
  T e[kQuad];
#pragma unroll
  for (int i = 0; i < kQuad; ++i) e[i] = from_f32<T>(v[i]);
  if (whole && left >= kQuad) {
    using B = typename Bits<T>::type;
    B raw;
    memcpy(&raw, e, sizeof(raw));
    *reinterpret_cast<B*>(at) = raw;
  } else {
#pragma unroll
    for (int i = 0; i < kQuad; ++i)
      if (i < left) at[i] = e[i];
  }
}

__device__ __forceinline__ float power_of_two(int e) { return __int_as_float((e + 127) << 23); }
__device__ __forceinline__ double power_of_two_f64(int e) { return __longlong_as_double((int64_t)(e + 1023) << 52); }

// The value in fp32 with the last bit set where it was not exact: rounding that to fewer bits is
// rounding the value itself, once.
__device__ __forceinline__ float to_odd(double x) {
  const float f = __double2float_rz(x);
  return static_cast<double>(f) == x ? f : __int_as_float(__float_as_int(f) | 1);
}
__device__ __forceinline__ bool finite(double x) { return fabs(x) <= DBL_MAX; }

// max over the warp's finite |x|, rounded up to fp32
__device__ __forceinline__ float largest(const double (&x)[kQuads][kQuad]) {
  float a = 0.0f;
#pragma unroll
  for (int u = 0; u < kQuads; ++u)
#pragma unroll
    for (int i = 0; i < kQuad; ++i)
      if (finite(x[u][i])) a = fmaxf(a, fminf(__double2float_ru(fabs(x[u][i])), FLT_MAX));
  return __uint_as_float(__reduce_max_sync(kFull, __float_as_uint(a)));
}
// smallest e with a <= 1.75 * 2^e
__device__ __forceinline__ int exponent_for(float a) {
  const uint32_t b = __float_as_uint(a);
  return static_cast<int>(b >> 23) - 127 + ((b & 0x7fffffu) > 0x600000u ? 1 : 0);
}
__device__ __forceinline__ int first_exponent(float a) { return min(max(exponent_for(a) - 8, kFirstLow), kHigh); }
__device__ __forceinline__ int second_exponent(float a) { return min(max(exponent_for(a), kSecondLow), kHigh); }

__device__ __forceinline__ uint32_t encode_first(const double (&x)[kQuad], double inv) {
  uint32_t w = 0;
#pragma unroll
  for (int i = 0; i < kQuad; i += 2) {
    const float2 f = make_float2(to_odd(x[i] * inv), to_odd(x[i + 1] * inv));
    uint32_t c = __nv_cvt_float2_to_fp8x2(f, __NV_SATFINITE, __NV_E4M3);
    if (!finite(x[i])) c |= 0x7fu;
    if (!finite(x[i + 1])) c |= 0x7f00u;
    w |= c << (8 * i);
  }
  return w;
}
__device__ __forceinline__ void decode_first(uint32_t w, float scale, float (&out)[kQuad]) {
#pragma unroll
  for (int i = 0; i < kQuad; i += 2) {
    const __half2 h = __half2(__nv_cvt_fp8x2_to_halfraw2(static_cast<__nv_fp8x2_storage_t>(w >> (8 * i)), __NV_E4M3));
    const float2 f = __half22float2(h);
    out[i] = f.x * scale;
    out[i + 1] = f.y * scale;
  }
}
// 2^-96 brings the held form's smallest normal value to fp32's, so its code is the upper bits of a
// (sub)normal fp32 value.
__device__ __forceinline__ uint32_t encode_second(const double (&x)[kQuad], double inv) {
  uint32_t w = 0;
#pragma unroll
  for (int i = 0; i < kQuad; ++i) {
    const uint32_t b = __float_as_uint(to_odd(fmin(x[i] * inv, 1.75) * 0x1p-96));
    uint32_t c = (b + 0x7ffffu + ((b >> 20) & 1u)) >> 20;
    if (c == 0 && x[i] > 0.0) c = 1;
    if (!finite(x[i])) c = 255;
    w |= c << (8 * i);
  }
  return w;
}
__device__ __forceinline__ void decode_second(uint32_t w, float scale, float (&out)[kQuad]) {
#pragma unroll
  for (int i = 0; i < kQuad; ++i) {
    const uint32_t c = (w >> (8 * i)) & 255u;
    out[i] = c == 255u ? __int_as_float(0x7fc00000) : __uint_as_float(c << 20) * 0x1p96f * scale;
  }
}

template <int kCap> __device__ __forceinline__ int tensor_of(const Table<kCap>& t, int chunk) {
  int lo = 0, hi = t.n - 1;  // the last tensor whose first chunk is not after this one
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (t.chunk[mid] <= chunk) lo = mid;
    else hi = mid - 1;
  }
  return lo;
}

template <typename P, typename G, bool k8, int kCap>
__global__ void __launch_bounds__(kThreads) adamw_kernel(const __grid_constant__ Table<kCap> t, Hyper h, State s) {
  __shared__ Rates sh_rates;
  __shared__ bool sh_last;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int chunks = t.chunk[t.n];
  int known = -1;
  for (int chunk = blockIdx.x; chunk < chunks; chunk += gridDim.x) {
    const int e = tensor_of(t, chunk);
    if (e != known) {
      known = e;
      __syncthreads();
      if (tid == 0) {
        const double n = static_cast<double>(s.steps[t.index[e]] + 1);
        const double lr = h.lr_device ? static_cast<double>(*h.lr_device) : h.lr;
        sh_rates.decay = static_cast<float>(1.0 - lr * h.weight_decay);
        sh_rates.step = static_cast<float>(lr / (1.0 - pow(h.beta1, n)));
        sh_rates.root = static_cast<float>(1.0 / sqrt(1.0 - pow(h.beta2, n)));
      }
      __syncthreads();
    }
    const Rates rate = sh_rates;
    const int64_t base = static_cast<int64_t>(chunk - t.chunk[e]) * kChunk + warp * kBlock;  // the warp's block
    if (base >= t.numel[e]) continue;
    const int64_t block = t.block[e] + base / kBlock;
    P* p = static_cast<P*>(t.param[e]) + base;
    const G* g = static_cast<const G*>(t.grad[e]) + base;
    const int64_t left = t.numel[e] - base;
    const bool p_whole = reinterpret_cast<uintptr_t>(p) % (kQuad * sizeof(P)) == 0;
    const bool g_whole = reinterpret_cast<uintptr_t>(g) % (kQuad * sizeof(G)) == 0;
    float pv[kQuads][kQuad], gv[kQuads][kQuad], mv[kQuads][kQuad], vv[kQuads][kQuad];
    if constexpr (k8) {
      const uint32_t* first = static_cast<uint32_t*>(s.first) + block * (kBlock / kQuad);
      const uint32_t* second = static_cast<uint32_t*>(s.second) + block * (kBlock / kQuad);
      const float fs = s.first_scale[block], ss = s.second_scale[block];
#pragma unroll
      for (int u = 0; u < kQuads; ++u) {
        decode_first(first[u * kWarp + lane], fs, mv[u]);
        decode_second(second[u * kWarp + lane], ss, vv[u]);
      }
    } else {
      const float* first = static_cast<float*>(s.first) + block * kBlock;
      const float* second = static_cast<float*>(s.second) + block * kBlock;
#pragma unroll
      for (int u = 0; u < kQuads; ++u) {
        load_quad(first + (u * kWarp + lane) * kQuad, kQuad, true, mv[u]);
        load_quad(second + (u * kWarp + lane) * kQuad, kQuad, true, vv[u]);
      }
    }
#pragma unroll
    for (int u = 0; u < kQuads; ++u) {
      const int at = (u * kWarp + lane) * kQuad;
      load_quad(p + at, left - at, p_whole, pv[u]);
      load_quad(g + at, left - at, g_whole, gv[u]);
    }
    if constexpr (k8) {
      double m[kQuads][kQuad], v[kQuads][kQuad];
#pragma unroll
      for (int u = 0; u < kQuads; ++u)
#pragma unroll
        for (int i = 0; i < kQuad; ++i) {
          const double gd = gv[u][i];
          m[u][i] = __dadd_rn(__dmul_rn(mv[u][i], h.beta1), __dmul_rn(gd, 1.0 - h.beta1));
          v[u][i] = __dadd_rn(__dmul_rn(vv[u][i], h.beta2), __dmul_rn(__dmul_rn(gd, gd), 1.0 - h.beta2));
          mv[u][i] = static_cast<float>(m[u][i]);
          vv[u][i] = static_cast<float>(v[u][i]);
        }
      const int fe = first_exponent(largest(m)), se = second_exponent(largest(v));
      uint32_t* first = static_cast<uint32_t*>(s.first) + block * (kBlock / kQuad);
      uint32_t* second = static_cast<uint32_t*>(s.second) + block * (kBlock / kQuad);
#pragma unroll
      for (int u = 0; u < kQuads; ++u) {
        first[u * kWarp + lane] = encode_first(m[u], power_of_two_f64(-fe));
        second[u * kWarp + lane] = encode_second(v[u], power_of_two_f64(-se));
      }
      if (lane == 0) {
        s.first_scale[block] = power_of_two(fe);
        s.second_scale[block] = power_of_two(se);
      }
    } else {
      const float b1 = static_cast<float>(h.beta1), a1 = static_cast<float>(1.0 - h.beta1);
      const float b2 = static_cast<float>(h.beta2), a2 = static_cast<float>(1.0 - h.beta2);
      float* first = static_cast<float*>(s.first) + block * kBlock;
      float* second = static_cast<float*>(s.second) + block * kBlock;
#pragma unroll
      for (int u = 0; u < kQuads; ++u) {
#pragma unroll
        for (int i = 0; i < kQuad; ++i) {
          mv[u][i] = fmaf(b1, mv[u][i], a1 * gv[u][i]);
          vv[u][i] = fmaf(b2, vv[u][i], a2 * gv[u][i] * gv[u][i]);
        }
        store_quad(first + (u * kWarp + lane) * kQuad, kQuad, true, mv[u]);
        store_quad(second + (u * kWarp + lane) * kQuad, kQuad, true, vv[u]);
      }
    }
#pragma unroll
    for (int u = 0; u < kQuads; ++u) {
#pragma unroll
      for (int i = 0; i < kQuad; ++i)
        pv[u][i] = fmaf(pv[u][i], rate.decay, -rate.step * (mv[u][i] / fmaf(sqrtf(vv[u][i]), rate.root, h.eps)));
      const int at = (u * kWarp + lane) * kQuad;
      store_quad(p + at, left - at, p_whole, pv[u]);
    }
  }
  // every block has read its step counts: the last one to come here advances them
  __syncthreads();
  if (tid == 0) {
    __threadfence();
    sh_last = atomicAdd(s.ticket, 1u) == gridDim.x - 1;
  }
  __syncthreads();
  if (!sh_last) return;
  for (int e = tid; e < t.n; e += kThreads) s.steps[t.index[e]] += 1;
  if (tid == 0) *s.ticket = 0;
}

__global__ void __launch_bounds__(kThreads) adamw_pack_kernel(const float* first, const float* second, int64_t blocks, State s) {
  const int lane = threadIdx.x & 31;
  const int64_t block = static_cast<int64_t>(blockIdx.x) * (kThreads / kWarp) + (threadIdx.x >> 5);
  if (block >= blocks) return;
  double m[kQuads][kQuad], v[kQuads][kQuad];
#pragma unroll
  for (int u = 0; u < kQuads; ++u) {
    float a[kQuad], b[kQuad];
    load_quad(first + block * kBlock + (u * kWarp + lane) * kQuad, kQuad, true, a);
    load_quad(second + block * kBlock + (u * kWarp + lane) * kQuad, kQuad, true, b);
#pragma unroll
    for (int i = 0; i < kQuad; ++i) m[u][i] = a[i], v[u][i] = b[i];
  }
  const int fe = first_exponent(largest(m)), se = second_exponent(largest(v));
#pragma unroll
  for (int u = 0; u < kQuads; ++u) {
    static_cast<uint32_t*>(s.first)[block * (kBlock / kQuad) + u * kWarp + lane] = encode_first(m[u], power_of_two_f64(-fe));
    static_cast<uint32_t*>(s.second)[block * (kBlock / kQuad) + u * kWarp + lane] = encode_second(v[u], power_of_two_f64(-se));
  }
  if (lane == 0) {
    s.first_scale[block] = power_of_two(fe);
    s.second_scale[block] = power_of_two(se);
  }
}

__global__ void __launch_bounds__(kThreads) adamw_unpack_kernel(State s, int64_t blocks, float* first, float* second) {
  const int lane = threadIdx.x & 31;
  const int64_t block = static_cast<int64_t>(blockIdx.x) * (kThreads / kWarp) + (threadIdx.x >> 5);
  if (block >= blocks) return;
  const float fs = s.first_scale[block], ss = s.second_scale[block];
#pragma unroll
  for (int u = 0; u < kQuads; ++u) {
    float a[kQuad], b[kQuad];
    decode_first(static_cast<const uint32_t*>(s.first)[block * (kBlock / kQuad) + u * kWarp + lane], fs, a);
    decode_second(static_cast<const uint32_t*>(s.second)[block * (kBlock / kQuad) + u * kWarp + lane], ss, b);
    store_quad(first + block * kBlock + (u * kWarp + lane) * kQuad, kQuad, true, a);
    store_quad(second + block * kBlock + (u * kWarp + lane) * kQuad, kQuad, true, b);
  }
}

int check_state(const mkg_adamw_state* s, int32_t bits, State* out) {
  MKG_REQUIRE(s && s->exp_avg && s->exp_avg_sq && s->steps && s->ticket, "adamw: null state");
  MKG_REQUIRE(bits == 32 || bits == 8, "adamw: moments in 32 or 8 bits, not %d", (int)bits);
  MKG_REQUIRE(bits == 32 || (s->exp_avg_scale && s->exp_avg_sq_scale), "adamw: moments in 8 bits need their scales");
  MKG_REQUIRE(s->total >= 0 && s->total % kBlock == 0 && s->total / kBlock < (int64_t(1) << 31),
              "adamw: %lld moments, not a multiple of %d below 2^39", (long long)s->total, kBlock);
  MKG_REQUIRE((reinterpret_cast<uintptr_t>(s->exp_avg) | reinterpret_cast<uintptr_t>(s->exp_avg_sq)) % 16 == 0,
              "adamw: moments must be 16-byte aligned");
  *out = State{s->exp_avg, s->exp_avg_sq, s->exp_avg_scale, s->exp_avg_sq_scale, s->steps, s->ticket};
  return MKG_OK;
}

template <typename P, typename G, bool k8, int kCap>
int launch(const Hyper& h, const State& s, int64_t n, void* const* params, const void* const* grads,
           const int64_t* numel, const int64_t* offset, const int64_t* index, cudaStream_t st) {
  int per_sm = 0;
  MKG_CUDA(cudaOccupancyMaxActiveBlocksPerMultiprocessor(&per_sm, adamw_kernel<P, G, k8, kCap>, kThreads, 0));
  const int64_t most = (int64_t)persistent_blocks(std::max(per_sm, 1));
  Table<kCap> t;
  for (int64_t i = 0; i < n;) {
    int64_t chunks = 0;
    t.n = 0;
    for (; i < n && t.n < kCap; ++i) {
      if (numel[i] == 0) continue;
      const int64_t more = (numel[i] + kChunk - 1) / kChunk;
      if (t.n > 0 && chunks + more > INT32_MAX - most) break;
      t.param[t.n] = params[i];
      t.grad[t.n] = grads[i];
      t.numel[t.n] = numel[i];
      t.block[t.n] = (int32_t)(offset[i] / kBlock);
      t.index[t.n] = (int32_t)index[i];
      t.chunk[t.n++] = (int32_t)chunks;
      chunks += more;
    }
    if (t.n == 0) return MKG_OK;
    t.chunk[t.n] = (int32_t)chunks;
    adamw_kernel<P, G, k8, kCap><<<(unsigned)std::min(chunks, most), kThreads, 0, st>>>(t, h, s);
    MKG_LAUNCHED("adamw_kernel");
  }
  return MKG_OK;
}

constexpr int kFew = 96, kMany = 800;

template <typename P, typename G, typename... A>
int by_size(int32_t bits, int64_t n, const Hyper& h, const State& s, A... a) {
  if (bits == 8) return n <= kFew ? launch<P, G, true, kFew>(h, s, n, a...) : launch<P, G, true, kMany>(h, s, n, a...);
  return n <= kFew ? launch<P, G, false, kFew>(h, s, n, a...) : launch<P, G, false, kMany>(h, s, n, a...);
}
template <typename P, typename... A> int by_grad(int32_t dtype, A... a) {
  switch (dtype) {
    case MKG_F32: return by_size<P, float>(a...);
    case MKG_BF16: return by_size<P, __nv_bfloat16>(a...);
    default: return by_size<P, __half>(a...);
  }
}

}  // namespace

int adamw_step(const mkg_adamw_params* p, const mkg_adamw_state* state, int64_t n, void* const* params,
               const void* const* grads, const int64_t* numel, const int64_t* offset, const int64_t* index,
               cudaStream_t st) {
  MKG_REQUIRE(p, "adamw_step: null parameters");
  MKG_REQUIRE(n >= 0 && (n == 0 || (params && grads && numel && offset && index)), "adamw_step: null argument");
  MKG_REQUIRE(p->param_dtype >= MKG_F32 && p->param_dtype <= MKG_F16 && p->grad_dtype >= MKG_F32 &&
                  p->grad_dtype <= MKG_F16, "adamw_step: unknown element type");
  MKG_REQUIRE(p->beta1 >= 0.0 && p->beta1 < 1.0 && p->beta2 >= 0.0 && p->beta2 < 1.0, "adamw_step: betas outside [0, 1)");
  MKG_REQUIRE(p->eps >= 0.0 && p->weight_decay >= 0.0 && (p->lr_device || p->lr >= 0.0),
              "adamw_step: lr, eps and weight_decay must not be negative");
  State s;
  if (int rc = check_state(state, p->state_bits, &s)) return rc;
  const int64_t size_p = p->param_dtype == MKG_F32 ? 4 : 2, size_g = p->grad_dtype == MKG_F32 ? 4 : 2;
  for (int64_t i = 0; i < n; ++i) {
    MKG_REQUIRE(numel[i] >= 0 && (numel[i] == 0 || (params[i] && grads[i])), "adamw_step: tensor %lld is null", (long long)i);
    MKG_REQUIRE(offset[i] >= 0 && offset[i] % kBlock == 0 && numel[i] <= state->total - offset[i],
                "adamw_step: tensor %lld outside the moments", (long long)i);
    MKG_REQUIRE(index[i] >= 0 && index[i] < state->tensors, "adamw_step: tensor %lld has no step count", (long long)i);
    MKG_REQUIRE(reinterpret_cast<uintptr_t>(params[i]) % size_p == 0 && reinterpret_cast<uintptr_t>(grads[i]) % size_g == 0,
                "adamw_step: tensor %lld is misaligned", (long long)i);
  }
  if (n == 0) return MKG_OK;
  const Hyper h{p->lr, p->beta1, p->beta2, p->weight_decay, (float)p->eps, p->lr_device};
  switch (p->param_dtype) {
    case MKG_F32: return by_grad<float>(p->grad_dtype, p->state_bits, n, h, s, params, grads, numel, offset, index, st);
    case MKG_BF16: return by_grad<__nv_bfloat16>(p->grad_dtype, p->state_bits, n, h, s, params, grads, numel, offset, index, st);
    default: return by_grad<__half>(p->grad_dtype, p->state_bits, n, h, s, params, grads, numel, offset, index, st);
  }
}

int adamw_pack(const mkg_adamw_state* state, const float* exp_avg, const float* exp_avg_sq, cudaStream_t st) {
  State s;
  if (int rc = check_state(state, 8, &s)) return rc;
  MKG_REQUIRE(exp_avg && exp_avg_sq && (reinterpret_cast<uintptr_t>(exp_avg) | reinterpret_cast<uintptr_t>(exp_avg_sq)) % 16 == 0,
              "adamw_pack: null or misaligned moments");
  const int64_t blocks = state->total / kBlock;
  if (blocks == 0) return MKG_OK;
  adamw_pack_kernel<<<(unsigned)((blocks + 7) / 8), kThreads, 0, st>>>(exp_avg, exp_avg_sq, blocks, s);
  MKG_LAUNCHED("adamw_pack_kernel");
  return MKG_OK;
}

int adamw_unpack(const mkg_adamw_state* state, float* exp_avg, float* exp_avg_sq, cudaStream_t st) {
  State s;
  if (int rc = check_state(state, 8, &s)) return rc;
  MKG_REQUIRE(exp_avg && exp_avg_sq && (reinterpret_cast<uintptr_t>(exp_avg) | reinterpret_cast<uintptr_t>(exp_avg_sq)) % 16 == 0,
              "adamw_unpack: null or misaligned moments");
  const int64_t blocks = state->total / kBlock;
  if (blocks == 0) return MKG_OK;
  adamw_unpack_kernel<<<(unsigned)((blocks + 7) / 8), kThreads, 0, st>>>(s, blocks, exp_avg, exp_avg_sq);
  MKG_LAUNCHED("adamw_unpack_kernel");
  return MKG_OK;
}

}  // namespace mkg
