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
// because the held values have the same relative spacing everywhere.  What is held is the fp64 sum
// rounded once: rounding to fp32 first would move about one sum in 10^6 to the neighbouring value, and
// with 16-bit gradients sums on the middle of two values are frequent (about one in 200).  The sums are
// taken in fp32 with a bound on their error; where both ends of the interval round to the same code that
// is the fp64 sum's code too, and only the others are taken again in fp64.  The update takes the fp32 sums.
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
// Blocks per SM.  fp32 moments: HBM-bound (20,624,575 fp32 values 85 us, 6.8 TB/s), 48 registers suffice.
// Moments in 8 bits: bound by instructions (about 80 a value) and their chains, 91 us for bf16 with 3 blocks,
// 96 with 4 (spills) and 108 with 2.
constexpr int kBlocks8 = 3, kBlocks32 = 5;
constexpr unsigned kFull = 0xffffffffu;
// Second moments below this, the largest held value less 1 in 14,000, do not saturate; larger ones are taken in fp64.
constexpr float kSecondClear = 0x1.bff8p120f;
constexpr int kFirstLow = -120, kFirstHigh = 119, kSecondLow = -90, kSecondHigh = 120;  // of the blocks' scales

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
  float plain_from;  // quotient()'s plain form from this eps on
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

template <typename T> __device__ __forceinline__ void spread(typename Bits<T>::type raw, float (&out)[kQuad]) {
  T e[kQuad];
  memcpy(e, &raw, sizeof(raw));
#pragma unroll
  for (int i = 0; i < kQuad; ++i) out[i] = to_f32<T>(e[i]);
}
template <typename T> __device__ __forceinline__ void load_quad(const T* at, float (&out)[kQuad]) {
  const typename Bits<T>::type raw = *reinterpret_cast<const typename Bits<T>::type*>(at);
  spread<T>(raw, out);
}
template <typename T> __device__ __forceinline__ void store_quad(T* at, const float (&v)[kQuad]) {
  T e[kQuad];
#pragma unroll
  for (int i = 0; i < kQuad; ++i) e[i] = from_f32<T>(v[i]);
  using B = typename Bits<T>::type;
  B raw;
  memcpy(&raw, e, sizeof(raw));
  *reinterpret_cast<B*>(at) = raw;
}
// A lane's share of a whole block as it is in memory, moments in 8 bits: what a warp loads for its next
// block while it works on this one.
template <typename G> struct Share {  // the parameters, needed last, are loaded when the block's turn comes
  typename Bits<G>::type g[kQuads];
  uint32_t first[kQuads], second[kQuads];
  float first_scale, second_scale;
};
// A lane's share of a block of a tensor: `left` values from `at` on exist, others read as 0.  whole: all
// 256 do, and `at` is aligned for loads of four.
template <typename T>
__device__ __forceinline__ void load_block(const T* at, int64_t left, bool whole, int lane, float (&out)[kQuads][kQuad]) {
  if (whole) {
#pragma unroll
    for (int u = 0; u < kQuads; ++u) load_quad(at + (u * kWarp + lane) * kQuad, out[u]);
  } else {
#pragma unroll
    for (int u = 0; u < kQuads; ++u)
#pragma unroll
      for (int i = 0; i < kQuad; ++i) {
        const int j = (u * kWarp + lane) * kQuad + i;
        out[u][i] = j < left ? to_f32<T>(at[j]) : 0.0f;
      }
  }
}
template <typename T>
__device__ __forceinline__ void store_block(T* at, int64_t left, bool whole, int lane, const float (&v)[kQuads][kQuad]) {
  if (whole) {
#pragma unroll
    for (int u = 0; u < kQuads; ++u) store_quad(at + (u * kWarp + lane) * kQuad, v[u]);
  } else {
#pragma unroll
    for (int u = 0; u < kQuads; ++u)
#pragma unroll
      for (int i = 0; i < kQuad; ++i) {
        const int j = (u * kWarp + lane) * kQuad + i;
        if (j < left) at[j] = from_f32<T>(v[u][i]);
      }
  }
}

__device__ __forceinline__ float power_of_two(int e) { return __int_as_float((e + 127) << 23); }
__device__ __forceinline__ double power_of_two_f64(int e) { return __longlong_as_double((int64_t)(e + 1023) << 52); }

// max that keeps a NaN (fmaxf drops it)
__device__ __forceinline__ float max_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}
// The value in fp32 with the last bit set where it was not exact: rounding that to fewer bits is
// rounding the value itself, once.
__device__ __forceinline__ float to_odd(double x) {
  const float f = __double2float_rz(x);
  return static_cast<double>(f) == x ? f : __int_as_float(__float_as_int(f) | 1);
}
__device__ __forceinline__ bool finite(double x) { return fabs(x) <= DBL_MAX; }

// smallest e with a <= 1.75 * 2^e: a mantissa above 0.75 carries into the exponent
__device__ __forceinline__ int exponent_for(float a) {
  return static_cast<int>((__float_as_uint(a) + 0x1fffffu) >> 23) - 127;
}
__device__ __forceinline__ int first_exponent(float a) { return min(max(exponent_for(a) - 8, kFirstLow), kFirstHigh); }
__device__ __forceinline__ int second_exponent(float a) { return min(max(exponent_for(a), kSecondLow), kSecondHigh); }
__device__ __forceinline__ float warp_max(float a) {  // of values >= 0
  return __uint_as_float(__reduce_max_sync(kFull, __float_as_uint(a)));
}
__device__ __forceinline__ float magnitude(double x) {  // |x| rounded up, as a block's largest counts it
  return finite(x) ? fminf(__double2float_ru(fabs(x)), FLT_MAX) : 0.0f;
}

// Codes of one moment, from fp64.
__device__ __forceinline__ uint32_t encode_first(double x, int e) {
  if (!finite(x)) return 0x7fu;
  return __nv_cvt_float_to_fp8(to_odd(x * power_of_two_f64(-e)), __NV_SATFINITE, __NV_E4M3);
}
// 2^-96 brings the held form's smallest normal value to fp32's, so its code is the upper bits of a
// (sub)normal fp32 value.
__device__ __forceinline__ uint32_t round_second(uint32_t b) { return (b + 0x7ffffu + ((b >> 20) & 1u)) >> 20; }
__device__ __forceinline__ uint32_t encode_second(double x, int e) {
  if (!finite(x)) return 255u;
  const uint32_t c = round_second(__float_as_uint(to_odd(fmin(x * power_of_two_f64(-e), 1.75) * 0x1p-96)));
  return c == 0 && x > 0.0 ? 1u : c;
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
__device__ __forceinline__ void decode_second(uint32_t w, float scale, float (&out)[kQuad]) {
  if (scale <= 0x1p30f) {
    const float s = scale * 0x1p96f;
#pragma unroll
    for (int i = 0; i < kQuad; ++i) out[i] = __uint_as_float(((w >> (8 * i)) & 255u) << 20) * s;
  } else {
#pragma unroll
    for (int i = 0; i < kQuad; ++i) out[i] = __uint_as_float(((w >> (8 * i)) & 255u) << 20) * 0x1p96f * scale;
  }
  if (((w & 0x7f7f7f7fu) + 0x01010101u) & w & 0x80808080u) {  // a byte of 255
#pragma unroll
    for (int i = 0; i < kQuad; ++i)
      if (((w >> (8 * i)) & 255u) == 255u) out[i] = __int_as_float(0x7fc00000);
  }
}

// A block's moments in 8 bits after a step, by one warp.
struct Held {
  uint32_t* first;   // the lane's words of the block, kWarp apart
  uint32_t* second;
  float* first_scale;
  float* second_scale;
};
// Both moments of one value in fp64, in the definition's order.
__device__ __forceinline__ double first_sum(const Hyper& h, float m, float g) {
  return __dadd_rn(__dmul_rn(m, h.beta1), __dmul_rn(g, 1.0 - h.beta1));
}
__device__ __forceinline__ double second_sum(const Hyper& h, float v, float g) {
  const double gd = g;
  return __dadd_rn(__dmul_rn(v, h.beta2), __dmul_rn(__dmul_rn(gd, gd), 1.0 - h.beta2));
}

// a's byte 3 of each word, words 0 to 3 as bytes 0 to 3
__device__ __forceinline__ uint32_t upper_bytes(const uint32_t (&t)[kQuad]) {
  return __byte_perm(__byte_perm(t[0], t[1], 0x0073), __byte_perm(t[2], t[3], 0x0073), 0x5410);
}
// 0x80 in every byte of w that is not 0
__device__ __forceinline__ uint32_t nonzero_bytes(uint32_t w) {
  return (((w & 0x7f7f7f7fu) + 0x7f7f7f7fu) | w) & 0x80808080u;
}

// m, v: the moments held before; they become the step's moments in fp32, and what is held of them is
// written.  g(u, i): the lane's gradients; again(q): the q-th of them once more, from memory.
template <typename Grad, typename Again>
__device__ __forceinline__ void step_held(const Hyper& h, const Held& at, float (&m)[kQuads][kQuad],
                                          float (&v)[kQuads][kQuad], float fs, float ss, Grad g, Again again,
                                          int lane) {
  const float b1 = static_cast<float>(h.beta1), a1 = static_cast<float>(1.0 - h.beta1);
  const float b2 = static_cast<float>(h.beta2), a2 = static_cast<float>(1.0 - h.beta2);
  float off[kQuads][kQuad];  // |fp32 sum - fp64 sum| of the first moment is below this
  float top1 = 0.0f, top2 = 0.0f, most_off = 0.0f;
#pragma unroll
  for (int u = 0; u < kQuads; ++u)
#pragma unroll
    for (int i = 0; i < kQuad; ++i) {
      const float x = b1 * m[u][i], y = a1 * g(u, i);
      m[u][i] = x + y;
      // b1, a1, both products and the sum are each off by 2^-24 of their size: 4 of them; twice that is allowed
      off[u][i] = fmaf(fabsf(x) + fabsf(y), 0x1p-21f, 0x1p-148f);
      v[u][i] = fmaf(b2, v[u][i], a2 * g(u, i) * g(u, i));
      top1 = max_nan(top1, fabsf(m[u][i]));
      most_off = fmaxf(most_off, off[u][i]);
      top2 = max_nan(top2, v[u][i]);
    }
  top1 = warp_max(top1);  // a NaN counts as the largest
  top2 = warp_max(top2);
  most_off = warp_max(most_off);
  int fe = first_exponent(top1 + most_off), se = second_exponent(top2 * (1.0f + 0x1p-20f));
  const bool clear = top1 <= FLT_MAX && top2 <= kSecondClear && first_exponent(fmaxf(top1 - most_off, 0.0f)) == fe &&
                     second_exponent(top2 * (1.0f - 0x1p-20f)) == se;
  uint32_t again1 = 0, again2 = 0;  // values to be taken in fp64: bit 7 - u of byte i
  uint32_t fw[kQuads], sw[kQuads];
  if (clear) {
    const float fi = power_of_two(-fe), si = power_of_two(-se);
#pragma unroll
    for (int u = 0; u < kQuads; ++u) {
      uint32_t lo[2], hi[2], t[kQuad];
#pragma unroll
      for (int i = 0; i < kQuad; i += 2) {
        const float d0 = off[u][i] * fi, d1 = off[u][i + 1] * fi, m0 = m[u][i], m1 = m[u][i + 1];
        lo[i / 2] = __nv_cvt_float2_to_fp8x2(make_float2(fmaf(m0, fi, -d0), fmaf(m1, fi, -d1)), __NV_SATFINITE, __NV_E4M3);
        hi[i / 2] = __nv_cvt_float2_to_fp8x2(make_float2(fmaf(m0, fi, d0), fmaf(m1, fi, d1)), __NV_SATFINITE, __NV_E4M3);
      }
      const uint32_t low = __byte_perm(lo[0], lo[1], 0x5410);
      fw[u] = __byte_perm(hi[0], hi[1], 0x5410);
      if (low != fw[u])  // the ends differ, and not as 0 and -0
        again1 |= (nonzero_bytes(low ^ fw[u]) & nonzero_bytes((low | fw[u]) & 0x7f7f7f7fu)) >> u;
      uint32_t near = 0xffffffffu;
#pragma unroll
      for (int i = 0; i < kQuad; ++i) {
        // the code in byte 3, rounded by the byte below it: v32 is off by at most 5 * 2^-24 of itself, 5 units
        // of its last place, and 16 of them around the middle go to fp64
        t[i] = __float_as_uint(v[u][i] * si * 0x1p-96f) * 16u + 0x800000u;
        near = min(near, t[i] * 256u + 0x10000u);
      }
      sw[u] = upper_bytes(t);
      if (near <= 0x20000u) {
#pragma unroll
        for (int i = 0; i < kQuad; ++i)
          if (t[i] * 256u + 0x10000u <= 0x20000u) again2 |= 0x80u << (8 * i) >> u;
      }
      if (nonzero_bytes(sw[u]) != 0x80808080u) {  // below the smallest held value: that, or 0 where nothing was added up
#pragma unroll
        for (int i = 0; i < kQuad; ++i)
          if (((sw[u] >> (8 * i)) & 255u) == 0 && (v[u][i] > 0.0f || again(u * kQuad + i) != 0.0f)) sw[u] |= 1u << (8 * i);
      }
    }
  } else {  // the block's largest values, exactly
    float high1 = 0.0f, high2 = 0.0f;
    again1 = again2 = 0xc0c0c0c0u;
#pragma unroll
    for (int u = 0; u < kQuads; ++u) {
      float om[kQuad], ov[kQuad];
      fw[u] = sw[u] = 0;
      decode_first(at.first[u * kWarp], fs, om);
      decode_second(at.second[u * kWarp], ss, ov);
#pragma unroll
      for (int i = 0; i < kQuad; ++i) {
        const float gi = again(u * kQuad + i);
        high1 = fmaxf(high1, magnitude(first_sum(h, om[i], gi)));
        high2 = fmaxf(high2, magnitude(second_sum(h, ov[i], gi)));
      }
    }
    fe = first_exponent(warp_max(high1));
    se = second_exponent(warp_max(high2));
  }
  // Every lane takes its own next value, so the warp goes round once for most blocks.  16-bit gradients
  // put a first moment on the middle of two values about once in 200.
  for (; again1; again1 &= again1 - 1) {
    const int bit = __ffs(again1) - 1, u = 7 - (bit & 7), to = bit & ~7;
    float old[kQuad];
    decode_first(at.first[u * kWarp] >> to, fs, old);
    const uint32_t code = encode_first(first_sum(h, old[0], again(u * kQuad + to / 8)), fe) << to;
#pragma unroll
    for (int w = 0; w < kQuads; ++w)
      if (w == u) fw[w] = (fw[w] & ~(255u << to)) | code;
  }
  for (; again2; again2 &= again2 - 1) {
    const int bit = __ffs(again2) - 1, u = 7 - (bit & 7), to = bit & ~7;
    float old[kQuad];
    decode_second(at.second[u * kWarp] >> to, ss, old);
    const uint32_t code = encode_second(second_sum(h, old[0], again(u * kQuad + to / 8)), se) << to;
#pragma unroll
    for (int w = 0; w < kQuads; ++w)
      if (w == u) sw[w] = (sw[w] & ~(255u << to)) | code;
  }
#pragma unroll
  for (int u = 0; u < kQuads; ++u) {
    at.first[u * kWarp] = fw[u];
    at.second[u * kWarp] = sw[u];
  }
  if (lane == 0) {
    *at.first_scale = power_of_two(fe);
    *at.second_scale = power_of_two(se);
  }
}

// m / (sqrt(v) r + eps) without the slow paths of sqrt and division for subnormal numbers, which moments
// that decay without a gradient reach (60,000,000 bf16 values took 395 us with them, 243 us without).
// Beside an eps of 2^-39 r or more a subnormal v counts as 0: its root is below 2^-63, its share of the sum
// below 2^-63 r, 2^-24 of eps.  r = 1 / sqrt(1 - b2^t) is largest at the first step, 31.6 for the usual 0.999;
// the form goes by that (by each tensor's own r, 20,624,575 bf16 values in 8 bits took 6 us more, in registers).
template <bool kPlain> __device__ __forceinline__ float quotient(float m, float v, float r, float eps) {
  float root, inv;
  if (kPlain) {
    asm("sqrt.approx.ftz.f32 %0, %1;" : "=f"(root) : "f"(v));
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(inv) : "f"(fmaf(root, r, eps)));
    return m * inv;
  }
  asm("sqrt.approx.f32 %0, %1;" : "=f"(root) : "f"(v));
  return __fdividef(m, fmaf(root, r, eps));
}

// b^n by squaring, off by about n units of 2^-53 of itself, which 1 - b^n does not see once b^n is small.  A
// block waits for it: pow and a division in fp64 kept the first chunk of each waiting for several us.
__device__ __forceinline__ double power(double b, int64_t n) {
  double r = 1.0;
  for (; n > 0; n >>= 1, b *= b)
    if (n & 1) r *= b;
  return r;
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
__global__ void __launch_bounds__(kThreads, k8 ? kBlocks8 : kBlocks32)
    adamw_kernel(const __grid_constant__ Table<kCap> t, Hyper h, State s, int run) {
  __shared__ Rates sh_rates[2];
  __shared__ bool sh_last;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int chunks = t.chunk[t.n];
  int known = -1, turn = 0;
  const bool plain = h.eps >= h.plain_from;
  Share<G> next;    // moments in 8 bits
  bool ready = false;  // next holds the block that comes
  const int end = min((static_cast<int>(blockIdx.x) + 1) * run, chunks);
  for (int chunk = blockIdx.x * run; chunk < end; ++chunk) {
    const int e = tensor_of(t, chunk);
    const bool fresh = e != known;
    if (fresh) {
      known = e;
      turn ^= 1;
      if (tid < 2) {  // the other warps need them only after their moments; the last ones may still be in use
        const double lr = h.lr_device ? static_cast<double>(*h.lr_device) : h.lr;
        const float left = static_cast<float>(1.0 - power(tid == 0 ? h.beta1 : h.beta2, s.steps[t.index[e]] + 1));
        if (tid == 0) {
          sh_rates[turn].decay = static_cast<float>(1.0 - lr * h.weight_decay);
          sh_rates[turn].step = static_cast<float>(lr) / left;
        } else {
          sh_rates[turn].root = 1.0f / sqrtf(left);
        }
      }
      __syncwarp();
    }
    const int64_t base = static_cast<int64_t>(chunk - t.chunk[e]) * kChunk + warp * kBlock;  // the warp's block
    const bool any = base < t.numel[e];
    const int64_t block = t.block[e] + base / kBlock;
    P* p = static_cast<P*>(t.param[e]) + base;
    const G* g = static_cast<const G*>(t.grad[e]) + base;
    const int64_t left = t.numel[e] - base;
    const bool whole = left >= kBlock && reinterpret_cast<uintptr_t>(p) % (kQuad * sizeof(P)) == 0 &&
                       reinterpret_cast<uintptr_t>(g) % (kQuad * sizeof(G)) == 0;
    float pv[kQuads][kQuad], gv[kQuads][kQuad], mv[kQuads][kQuad], vv[kQuads][kQuad];
    float fs = 0.0f, ss = 0.0f;
    if constexpr (k8) {
      if (any) {
        const uint32_t* first = static_cast<uint32_t*>(s.first) + block * (kBlock / kQuad) + lane;
        const uint32_t* second = static_cast<uint32_t*>(s.second) + block * (kBlock / kQuad) + lane;
        auto fetch = [&](int64_t ahead) {  // `ahead` blocks further on
#pragma unroll
          for (int u = 0; u < kQuads; ++u) {
            const int64_t j = ahead * kBlock + (u * kWarp + lane) * kQuad;
            next.g[u] = *reinterpret_cast<const typename Bits<G>::type*>(g + j);
            next.first[u] = first[ahead * (kBlock / kQuad) + u * kWarp];
            next.second[u] = second[ahead * (kBlock / kQuad) + u * kWarp];
          }
          next.first_scale = s.first_scale[block + ahead];
          next.second_scale = s.second_scale[block + ahead];
        };
        if (whole) {
          load_block(p, left, true, lane, pv);
          if (!ready) fetch(0);
          fs = next.first_scale;
          ss = next.second_scale;
#pragma unroll
          for (int u = 0; u < kQuads; ++u) {
            spread<G>(next.g[u], gv[u]);
            decode_first(next.first[u], fs, mv[u]);
            decode_second(next.second[u], ss, vv[u]);
          }
          // the same warp's block of the next chunk, if that is whole and the same tensor's
          ready = chunk + 1 < end && left - kChunk >= kBlock;
          if (ready) fetch(kChunk / kBlock);
        } else {
          ready = false;
          fs = s.first_scale[block];
          ss = s.second_scale[block];
#pragma unroll
          for (int u = 0; u < kQuads; ++u) {
            decode_first(first[u * kWarp], fs, mv[u]);
            decode_second(second[u * kWarp], ss, vv[u]);
          }
          load_block(p, left, false, lane, pv);
          load_block(g, left, false, lane, gv);
        }
      }
    }
    if (any) {
      if constexpr (!k8) {
        const float* first = static_cast<float*>(s.first) + block * kBlock;
        const float* second = static_cast<float*>(s.second) + block * kBlock;
        load_block(first, kBlock, true, lane, mv);
        load_block(second, kBlock, true, lane, vv);
        load_block(p, left, whole, lane, pv);
        load_block(g, left, whole, lane, gv);
      }
      if constexpr (k8) {
        const Held at{static_cast<uint32_t*>(s.first) + block * (kBlock / kQuad) + lane,
                      static_cast<uint32_t*>(s.second) + block * (kBlock / kQuad) + lane, s.first_scale + block,
                      s.second_scale + block};
        step_held(
            h, at, mv, vv, fs, ss, [&](int u, int i) { return gv[u][i]; },
            [&](int q) {
              const int j = (q / kQuad * kWarp + lane) * kQuad + q % kQuad;
              return j < left ? to_f32<G>(g[j]) : 0.0f;
            },
            lane);
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
        }
        store_block(first, kBlock, true, lane, mv);
        store_block(second, kBlock, true, lane, vv);
      }
    }
    if (fresh) __syncthreads();
    if (!any) continue;
    const Rates rate = sh_rates[turn];
#pragma unroll
    for (int u = 0; u < kQuads; ++u) {
#pragma unroll
      for (int i = 0; i < kQuad; ++i)
        pv[u][i] = fmaf(pv[u][i], rate.decay,
                        -rate.step * (plain ? quotient<true>(mv[u][i], vv[u][i], rate.root, h.eps)
                                            : quotient<false>(mv[u][i], vv[u][i], rate.root, h.eps)));
    }
    store_block(p, left, whole, lane, pv);
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
  float m[kQuads][kQuad], v[kQuads][kQuad], a = 0.0f, b = 0.0f;
#pragma unroll
  for (int u = 0; u < kQuads; ++u) {
    load_quad(first + block * kBlock + (u * kWarp + lane) * kQuad, m[u]);
    load_quad(second + block * kBlock + (u * kWarp + lane) * kQuad, v[u]);
#pragma unroll
    for (int i = 0; i < kQuad; ++i) {
      a = fmaxf(a, magnitude(m[u][i]));
      b = fmaxf(b, magnitude(v[u][i]));
    }
  }
  const int fe = first_exponent(warp_max(a)), se = second_exponent(warp_max(b));
#pragma unroll
  for (int u = 0; u < kQuads; ++u) {
    uint32_t fw = 0, sw = 0;
#pragma unroll
    for (int i = 0; i < kQuad; ++i) {
      fw |= encode_first(m[u][i], fe) << (8 * i);
      sw |= encode_second(v[u][i], se) << (8 * i);
    }
    static_cast<uint32_t*>(s.first)[block * (kBlock / kQuad) + u * kWarp + lane] = fw;
    static_cast<uint32_t*>(s.second)[block * (kBlock / kQuad) + u * kWarp + lane] = sw;
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
    store_quad(first + block * kBlock + (u * kWarp + lane) * kQuad, a);
    store_quad(second + block * kBlock + (u * kWarp + lane) * kQuad, b);
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
  cudaFuncAttributes loaded;  // loads the kernel: a call without values prepares a capture
  MKG_CUDA(cudaFuncGetAttributes(&loaded, adamw_kernel<P, G, k8, kCap>));
  Table<kCap> t;
  for (int64_t i = 0; i < n;) {
    int64_t chunks = 0;
    t.n = 0;
    for (; i < n && t.n < kCap; ++i) {
      if (numel[i] == 0) continue;
      const int64_t more = (numel[i] + kChunk - 1) / kChunk;
      if (t.n > 0 && chunks + more > INT32_MAX / 2) break;
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
    // Four chunks of a block share what a tensor's rates cost, as long as there are blocks enough for every
    // SM several times over: 60,000,000 bf16 values took 301 us with runs of 1, 243 us with 4 and 255 us with
    // 16, and 27 tensors of 219,815 values 7 us with 1 and 13 us with 4.
    const int run = chunks >= persistent_blocks(8) * 4 ? 4 : 1;
    adamw_kernel<P, G, k8, kCap><<<(unsigned)((chunks + run - 1) / run), kThreads, 0, st>>>(t, h, s, run);
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
  const float plain_from = (float)(0x1p-39 / std::sqrt(1.0 - p->beta2));
  const Hyper h{p->lr, p->beta1, p->beta2, p->weight_decay, (float)p->eps, plain_from, p->lr_device};
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
