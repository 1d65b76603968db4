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

#include "mkg_common.cuh"
#include "mkg_internal.h"

namespace mkg {
namespace {

constexpr float kLn2 = 0.693147180559945309f;
constexpr float kInf = __builtin_inff();
constexpr int kTopMax = MKG_LOGPROB_TOPK_MAX;
// Threads per SM that stream rows.  64 registers each hold a round of loads without spilling; with
// alternatives and no mask 42 do, and more blocks stream while others order theirs (227 -> 211 us on 64
// rows of 4,594,485 fp32 logits).
constexpr int kResident = 1024, kResidentTop = 1536;
constexpr int kNarrowThreads = 64;   // two rows, a warp each
constexpr int64_t kNarrow = 2040;    // rows up to this width are held by one warp: 64 values a lane, wherever they start
constexpr int64_t kManyRows = 4096;  // enough to fill the SMs with a warp or a block each
constexpr int kCand = 256;           // alternatives collected before they are ordered
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
// Two fp32 values in one register pair: sm_100 adds, multiplies and fuses them in one instruction.
using Pair = unsigned long long;
__device__ __forceinline__ Pair pack2(float a, float b) {
  Pair r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ void unpack2(Pair p, float& a, float& b) { asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(p)); }
__device__ __forceinline__ Pair add2(Pair a, Pair b) {
  Pair r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ Pair mul2(Pair a, Pair b) {
  Pair r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ Pair fma2(Pair a, Pair b, Pair c) {
  Pair r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
// y = (x - m) c with -inf brought to where 2^y is 0 but y stays finite (0 * y must be 0)
__device__ __forceinline__ float scaled(float x, float m, float c) { return max_nan((x - m) * c, -256.0f); }

template <typename T> constexpr int kVec = 16 / sizeof(T);
constexpr int kUnroll = 4;  // 16-byte loads in flight per thread

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

  __device__ __forceinline__ bool whole(int slot) const { return first(slot) >= 0 && first(slot) + kVec<T> <= width; }

  // a slot that lies in the row, as it is in memory: its logits and its candidates' bytes
  struct Raw {
    uint4 x;
    uint2 on;
  };
  template <bool kMask> __device__ __forceinline__ Raw fetch(int slot) const {
    const int j0 = first(slot);
    Raw w;
    w.x = __ldg(reinterpret_cast<const uint4*>(x + j0));
    if constexpr (kMask) {
      if (mask_vec) {
        if constexpr (kVec<T> == 4) w.on.x = __ldg(reinterpret_cast<const uint32_t*>(mask + j0));
        else w.on = __ldg(reinterpret_cast<const uint2*>(mask + j0));
      } else {
        uint8_t on[8];
#pragma unroll
        for (int i = 0; i < kVec<T>; ++i) on[i] = __ldg(mask + j0 + i);
        memcpy(&w.on, on, 8);
      }
    }
    return w;
  }
  // in fp32, non-candidates as -inf
  template <bool kMask> __device__ __forceinline__ void values(const Raw& w, float (&v)[kVec<T>]) const {
    T e[kVec<T>];
    memcpy(e, &w.x, 16);
#pragma unroll
    for (int i = 0; i < kVec<T>; ++i) v[i] = to_f32<T>(e[i]);
    if constexpr (kMask) {
#pragma unroll
      for (int i = 0; i < kVec<T>; ++i)
        if (((i < 4 ? w.on.x : w.on.y) >> (8 * (i & 3)) & 255u) == 0) v[i] = -kInf;
    }
  }
  // any slot; columns outside the row as -inf
  template <bool kMask> __device__ __forceinline__ void load(int slot, float (&v)[kVec<T>]) const {
    if (whole(slot)) return values<kMask>(fetch<kMask>(slot), v);
    const int j0 = first(slot);
#pragma unroll
    for (int i = 0; i < kVec<T>; ++i) {
      const int j = j0 + i;
      const bool in = j >= 0 && j < width && (!kMask || __ldg(mask + j) != 0);
      v[i] = in ? to_f32<T>(x[j]) : -kInf;
    }
  }
};

// Hands a thread its slots of [lo, hi), kT apart and in ascending order: whole ones in rounds of up to
// kUnroll, all of a round's loads before its first use, and those that reach over the row's ends one by
// one.  many(slot, n, full): n slots from `slot` on; full: n is kUnroll.
template <typename T, int kT, typename Many, typename One>
__device__ __forceinline__ void for_slots(const RowView<T>& view, int lo, int hi, int tid, Many many, One one) {
  int slot = lo + tid;
  if (slot < hi && !view.whole(slot)) {
    one(slot);
    slot += kT;
  }
  const int inner = hi == view.slots && hi > lo && !view.whole(hi - 1) ? hi - 1 : hi;
  for (; slot + (kUnroll - 1) * kT < inner; slot += kUnroll * kT) many(slot, kUnroll, std::true_type());
  if (slot < inner) {
    const int n = (inner - slot + kT - 1) / kT;
    many(slot, n, std::false_type());
    slot += n * kT;
  }
  if (slot < hi) one(slot);
}

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
// The keys of every kLanes lanes of a warp in ascending order of the lanes.
template <int kLanes = kWarp>
__device__ __forceinline__ unsigned long long sort_ascending(unsigned long long v, int lane) {
#pragma unroll
  for (int size = 2; size <= kLanes; size <<= 1)
#pragma unroll
    for (int o = size >> 1; o > 0; o >>= 1)
      v = exchange(v, o, ((lane & o) != 0) == ((lane & size) == 0 || size == kLanes));
  return v;
}
// `best` descending over kLanes lanes, `add` ascending: the kLanes largest of both, descending.
template <int kLanes = kWarp>
__device__ __forceinline__ unsigned long long merge_best(unsigned long long best, unsigned long long add, int lane) {
  unsigned long long v = best > add ? best : add;
#pragma unroll
  for (int o = kLanes / 2; o > 0; o >>= 1) v = exchange(v, o, (lane & o) == 0);
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

// One given column of a row: what log p needs of it, read before the row is streamed so that the two
// dependent loads are not waited for at the end.
struct Target {
  float x;    // its logit
  int state;  // 0: padding, 1: a candidate, 2: none, 3: outside the row
};
template <typename T>
__device__ __forceinline__ Target read_target(const Rows& r, const int64_t* targets, int64_t row, int q, const T* x,
                                              const uint8_t* mask) {
  Target t{0.0f, 0};
  if (q >= r.targets) return t;
  const int64_t id = targets[row * r.targets + q];
  if (id < -1 || id >= r.width) t.state = 3;
  else if (id >= 0) {
    t.state = mask == nullptr || mask[id] != 0 ? 1 : 2;
    t.x = to_f32<T>(x[id]);
  }
  return t;
}

// The outputs of one row by the threads of a warp or block (`first` of `count`); `mine`: the thread's
// first target; `best`: the row's largest keys, descending over the lanes of the first warp.
template <typename T>
__device__ __forceinline__ void finish_row(const Rows& r, const Outputs& o, int64_t row, const T* x,
                                           const uint8_t* mask, const int64_t* targets, Target mine, Moments a,
                                           unsigned long long best, int first, int count) {
  const bool none = a.m == -kInf && a.s == 0.0f;
  const float log2s = none ? -kInf : a.s == a.s ? log2f(a.s) : a.s;
  if (first == 0) {
    o.lse[row] = none ? -kInf : fmaf(log2s, kLn2, a.m * r.inv_tau) + (a.s - a.s);
    o.entropy[row] = none ? 0.0f : fmaxf(kLn2 * (log2s - a.t / a.s), 0.0f) + (a.s - a.s);
    if (o.stats) {
      o.stats[2 * row] = a.m;
      o.stats[2 * row + 1] = a.s;
    }
  }
  for (int q = first; q < r.targets; q += count) {
    if (q != first) mine = read_target<T>(r, targets, row, q, x, mask);
    float lp = 0.0f;
    if (mine.state == 3) {
      raise_flag(o.err, MKG_DEV_BAD_TARGET);
      lp = __int_as_float(0x7fc00000);
    } else if (mine.state != 0) {
      lp = none ? -kInf : mine.state == 2 ? -kInf + (a.s - a.s) : kLn2 * ((mine.x - a.m) * r.c - log2s);
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

// ---------------------------------------------------------------- the largest keys of a warp or block
// The topk-th largest of one key per thread of the block, 0 if there are fewer; sh: a key per thread.
template <int kWarps>
__device__ __forceinline__ unsigned long long floor_of(unsigned long long mine, int topk, unsigned long long* sh) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  unsigned long long v = sort_ascending(mine, lane);
  unsigned long long best = __shfl_sync(kFull, v, 31 - lane);
#pragma unroll
  for (int half = kWarps / 2; half > 0; half >>= 1) {  // the upper half of the warps hands its 32 to the lower
    if (warp >= half && warp < 2 * half) sh[warp * kWarp + (31 - lane)] = best;
    __syncthreads();
    if (warp < half) best = merge_best(best, sh[(warp + half) * kWarp + lane], lane);
    __syncthreads();
  }
  if (threadIdx.x == topk - 1) sh[0] = best;
  __syncthreads();
  return sh[0];
}
// The warp's part of a list of keys in shared memory, merged into `best`.
__device__ __forceinline__ unsigned long long merge_list(unsigned long long best, const unsigned long long* list, int n,
                                                         int lane) {
  for (int i = 0; i < n; i += kWarp)
    best = merge_best(best, sort_ascending(i + lane < n ? list[i + lane] : 0, lane), lane);
  return best;
}

// ---------------------------------------------------------------- narrow rows: a warp, or eight lanes each
// Rows of about a hundred columns keep only a quarter of a warp busy with columns, and what a row costs
// besides (sums over the lanes, ordering, outputs: about 800 instructions of a warp) is shared by four of
// them: 65,536 rows of 103 fp32 logits with 5 alternatives took 60 us forward and 53 us backward with a
// warp each, 29 and 25 us with eight lanes.
template <int kLanes> __device__ __forceinline__ float lanes_max(float v) {
#pragma unroll
  for (int o = kLanes / 2; o > 0; o >>= 1) v = fmaxf(v, __shfl_xor_sync(kFull, v, o));
  return v;
}
template <int kLanes> __device__ __forceinline__ float lanes_sum(float v) {
#pragma unroll
  for (int o = kLanes / 2; o > 0; o >>= 1) v += __shfl_xor_sync(kFull, v, o);
  return v;
}

// The kLanes largest keys of each row of a warp, descending over its lanes, from its n candidates in shared
// memory; more than fit (a few lanes hold many of the largest): from the row itself, merged as it comes.
template <typename T, bool kMask, int kLanes>
__device__ __forceinline__ unsigned long long order_lanes(const unsigned long long* cand, int n, int room,
                                                          const Rows& r, const T* x, const uint8_t* mask, int lane,
                                                          int part) {
  __syncwarp();
  unsigned long long best = 0;
  const int most = __reduce_max_sync(kFull, n);
  if (most <= room) {
    for (int i = 0; i < most; i += kLanes)
      best = merge_best<kLanes>(best, sort_ascending<kLanes>(i + part < n ? cand[i + part] : 0, lane), lane);
  } else {
    for (int j = part; j < ((r.width + kLanes - 1) & -kLanes); j += kLanes) {
      const float w = j < r.width && (!kMask || mask[j] != 0) ? to_f32<T>(x[j]) : -kInf;
      const unsigned long long k = w > -kInf ? rank_key(w, static_cast<uint32_t>(j)) : 0;
      if (__any_sync(kFull, k > __shfl_sync(kFull, best, lane - part + r.topk - 1)))
        best = merge_best<kLanes>(best, sort_ascending<kLanes>(k, lane), lane);
    }
  }
  return best;
}

template <typename T, bool kMask, int kSlots, int kLanes>
__global__ void __launch_bounds__(kNarrowThreads) logprob_narrow_kernel(Rows r, const T* __restrict__ logits,
                                                                        const uint8_t* __restrict__ masks,
                                                                        const int64_t* __restrict__ targets, Outputs o) {
  constexpr int kRows = kNarrowThreads / kLanes, kRoom = 2 * kLanes;
  __shared__ unsigned long long sh_cand[kRows][kRoom];
  const int lane = threadIdx.x & 31, part = lane % kLanes, own = threadIdx.x / kLanes;
  int64_t row = static_cast<int64_t>(blockIdx.x) * kRows + own;
  if (row - lane / kLanes >= r.rows) return;  // the whole warp is past the end
  const bool valid = row < r.rows;  // others of the warp repeat the last row and write nothing
  row = min(row, r.rows - 1);
  const T* x = logits + row * r.stride;
  const uint8_t* mask = kMask ? masks + row * r.mask_stride : nullptr;
  const RowView<T> view(x, mask, r.width);
  const Target target = read_target<T>(r, targets, row, part, x, mask);
  float v[kSlots][kVec<T>];
#pragma unroll
  for (int q = 0; q < kSlots; ++q) {
    const int slot = q * kLanes + part;
    if (slot < view.slots) {
      view.template load<kMask>(slot, v[q]);
    } else {
#pragma unroll
      for (int i = 0; i < kVec<T>; ++i) v[q][i] = -kInf;
    }
  }
  Moments a{-kInf, 0.0f, 0.0f};
  int at = 0;  // the column where the lane first met its largest
#pragma unroll
  for (int q = 0; q < kSlots; ++q)
#pragma unroll
    for (int i = 0; i < kVec<T>; ++i)
      if (v[q][i] > a.m) {
        a.m = v[q][i];
        at = view.first(q * kLanes + part) + i;
      }
  const unsigned long long mine = a.m > -kInf ? rank_key(a.m, static_cast<uint32_t>(at)) : 0;
  a.m = lanes_max<kLanes>(a.m);
  const float from = a.m == -kInf ? 0.0f : a.m;
#pragma unroll
  for (int q = 0; q < kSlots; ++q)
#pragma unroll
    for (int i = 0; i < kVec<T>; ++i) {
      const float y = scaled(v[q][i], from, r.c);
      const float e = ex2(y);
      a.s += e;
      a.t = fmaf(e, y, a.t);
    }
  a.s = lanes_sum<kLanes>(a.s);
  a.t = lanes_sum<kLanes>(a.t);
  unsigned long long best = 0;
  if (r.topk > 0) {
    // elements below the topk-th largest of the lanes' maxima have topk better ones
    const unsigned long long sorted = sort_ascending<kLanes>(mine, lane);
    const unsigned long long floor = __shfl_sync(kFull, sorted, lane - part + kLanes - r.topk);
    const float least = floor ? packed_value(floor) : -kInf;
    const int least_at = floor ? static_cast<int>(packed_rank(floor)) : 0x7fffffff;
    unsigned long long* cand = sh_cand[own];
    const unsigned before = ((1u << part) - 1) << (lane - part);  // the row's lanes before this one
    const unsigned row_lanes = (kLanes == kWarp ? kFull : (1u << (kLanes & 31)) - 1) << (lane - part);
    int n = 0;
#pragma unroll
    for (int q = 0; q < kSlots; ++q)
#pragma unroll
      for (int i = 0; i < kVec<T>; ++i) {
        const int j = view.first(q * kLanes + part) + i;
        const bool in = v[q][i] > least || (v[q][i] == least && v[q][i] > -kInf && j <= least_at);
        const unsigned who = __ballot_sync(kFull, in);
        const int to = n + __popc(who & before);
        if (in && to < kRoom) cand[to] = rank_key(v[q][i], static_cast<uint32_t>(j));
        n += __popc(who & row_lanes);
      }
    best = order_lanes<T, kMask, kLanes>(cand, n, kRoom, r, x, mask, lane, part);
  }
  if (valid) finish_row<T>(r, o, row, x, mask, targets, target, a, best, part, kLanes);
}

// ---------------------------------------------------------------- wider rows: blocks, joined if several
struct Partial {
  float m, s, t, pad;
};

// Joins the warps' (m, s, t) of a block; every thread gets the result.
template <int kWarps> __device__ __forceinline__ Moments block_join(Moments a, float c, Moments* sh) {
  const int lane = threadIdx.x & 31;
  a = warp_join(a, c);
  if (lane == 0) sh[threadIdx.x >> 5] = a;
  __syncthreads();
  return warp_join(lane < kWarps ? sh[lane] : Moments{-kInf, 0.0f, 0.0f}, c);
}

// A thread's share of a row while it streams: the largest element and where it was first met, and the
// sums seen from `ref`.  ref follows m only when 2^y would pass 2^kMargin: in a warp some lane meets a
// new maximum in most rounds, and rescaling each time took half of the loop's instructions.
constexpr float kMargin = 8.0f;
struct Stream {
  float m, ref, limit;  // limit = ref + kMargin / c
  int at;
  Pair s, t;
};
template <typename T> __device__ __forceinline__ void consume(const float (&v)[kVec<T>], int slot, float c, Stream& a) {
  float big = v[0];
#pragma unroll
  for (int i = 1; i < kVec<T>; ++i) big = fmaxf(big, v[i]);
  if (big > a.m) {
    a.m = big;
    a.at = slot;
  }
  if (big > a.limit) {
    float s0, s1, t0, t1;
    unpack2(a.s, s0, s1);
    unpack2(a.t, t0, t1);
    Moments lo{a.ref, s0, t0}, hi{a.ref, s1, t1};
    shift_to(lo, big, c);
    shift_to(hi, big, c);
    a.s = pack2(lo.s, hi.s);
    a.t = pack2(lo.t, hi.t);
    a.ref = big;
    a.limit = big + kMargin / c;
  }
  const float from = a.ref == -kInf ? 0.0f : a.ref;
  const Pair from2 = pack2(-from, -from), c2 = pack2(c, c);
#pragma unroll
  for (int i = 0; i < kVec<T>; i += 2) {
    float y0, y1;
    unpack2(mul2(add2(pack2(v[i], v[i + 1]), from2), c2), y0, y1);
    y0 = max_nan(y0, -256.0f);
    y1 = max_nan(y1, -256.0f);
    const Pair e = pack2(ex2(y0), ex2(y1));
    a.s = add2(a.s, e);
    a.t = fma2(e, pack2(y0, y1), a.t);
  }
}

// A thread's slots of [lo, hi), kT apart: its moments, and the key of its largest element and the slot where
// that was first met (0: no candidate).
template <typename T, bool kMask, int kT>
__device__ __forceinline__ unsigned long long stream_slots(const RowView<T>& view, int lo, int hi, int tid, float c,
                                                           Moments& a) {
  Stream own{-kInf, -kInf, -kInf, 0, 0, 0};
  for_slots<T, kT>(
      view, lo, hi, tid,
      [&](int slot, int n, auto full) {
        typename RowView<T>::Raw raw[kUnroll];
#pragma unroll
        for (int u = 0; u < kUnroll; ++u)
          if (full || u < n) raw[u] = view.template fetch<kMask>(slot + u * kT);
#pragma unroll
        for (int u = 0; u < kUnroll; ++u) {
          if (!full && u >= n) break;
          float v[kVec<T>];
          view.template values<kMask>(raw[u], v);
          consume<T>(v, slot + u * kT, c, own);
        }
      },
      [&](int slot) {
        float v[kVec<T>];
        view.template load<kMask>(slot, v);
        consume<T>(v, slot, c, own);
      });
  float s0, s1, t0, t1;
  unpack2(own.s, s0, s1);
  unpack2(own.t, t0, t1);
  a = {own.ref, s0 + s1, t0 + t1};
  shift_to(a, own.m, c);
  a.m = own.m;
  return a.m > -kInf ? rank_key(a.m, static_cast<uint32_t>(own.at)) : 0;
}

// Many rows that a warp streams each, or eight lanes: no registers hold the row, so 32 to 40 warps an SM hide
// the loads, and nothing waits at a barrier.  Alternatives as in a block: the best lanes' slots again (from L1 or
// L2).
constexpr int kStreamThreads = 128;
template <typename T, bool kMask, int kLanes>
__global__ void __launch_bounds__(kStreamThreads, kMask ? 8 : 10)
    logprob_stream_kernel(Rows r, const T* __restrict__ logits, const uint8_t* __restrict__ masks,
                          const int64_t* __restrict__ targets, Outputs o) {
  constexpr int kRows = kStreamThreads / kLanes, kRoom = 2 * kLanes;
  __shared__ unsigned long long sh_cand[kRows][kRoom];
  __shared__ int sh_winner[kRows][kLanes];
  const int lane = threadIdx.x & 31, part = lane % kLanes, own = threadIdx.x / kLanes;
  int64_t row = static_cast<int64_t>(blockIdx.x) * kRows + own;
  if (row - lane / kLanes >= r.rows) return;  // the whole warp is past the end
  const bool valid = row < r.rows;  // others of the warp repeat the last row and write nothing
  row = min(row, r.rows - 1);
  const T* x = logits + row * r.stride;
  const uint8_t* mask = kMask ? masks + row * r.mask_stride : nullptr;
  const RowView<T> view(x, mask, r.width);
  const Target target = read_target<T>(r, targets, row, part, x, mask);
  Moments a;
  const unsigned long long mine = stream_slots<T, kMask, kLanes>(view, 0, view.slots, part, r.c, a);
  const float M = lanes_max<kLanes>(a.m);
  shift_to(a, M, r.c);
  a = {M, lanes_sum<kLanes>(a.s), lanes_sum<kLanes>(a.t)};
  unsigned long long best = 0;
  if (r.topk > 0) {
    const unsigned long long sorted = sort_ascending<kLanes>(mine, lane);
    const unsigned long long floor = __shfl_sync(kFull, sorted, lane - part + kLanes - r.topk);
    const float least = floor ? packed_value(floor) : -kInf;
    const uint32_t least_slot = floor ? packed_rank(floor) : 0xffffffffu;
    const unsigned before = ((1u << part) - 1) << (lane - part);  // the row's lanes before this one
    const unsigned row_lanes = (kLanes == kWarp ? kFull : (1u << (kLanes & 31)) - 1) << (lane - part);
    const bool winner = mine != 0 && mine >= floor;
    const unsigned winners = __ballot_sync(kFull, winner) & row_lanes;
    if (winner) sh_winner[own][__popc(winners & before)] = part;
    __syncwarp();
    const int per = (view.slots + kLanes - 1) / kLanes;  // slots of a lane
    const int pairs = __popc(winners) * per;
    const int most_pairs = __reduce_max_sync(kFull, pairs);
    unsigned long long* cand = sh_cand[own];
    int n = 0;
    for (int q = part; q < ((most_pairs + kLanes - 1) & -kLanes); q += kLanes) {
      const int slot = q < pairs ? sh_winner[own][q / per] + q % per * kLanes : view.slots;
      float v[kVec<T>];
      if (slot < view.slots) {
        view.template load<kMask>(slot, v);
      } else {
#pragma unroll
        for (int i = 0; i < kVec<T>; ++i) v[i] = -kInf;
      }
#pragma unroll
      for (int i = 0; i < kVec<T>; ++i) {
        const bool in = v[i] > least || (v[i] == least && v[i] > -kInf && static_cast<uint32_t>(slot) <= least_slot);
        const unsigned who = __ballot_sync(kFull, in);
        if (who == 0) continue;
        const int to = n + __popc(who & before);
        if (in && to < kRoom) cand[to] = rank_key(v[i], static_cast<uint32_t>(view.first(slot) + i));
        n += __popc(who & row_lanes);
      }
    }
    best = order_lanes<T, kMask, kLanes>(cand, n, kRoom, r, x, mask, lane, part);
  }
  if (valid) finish_row<T>(r, o, row, x, mask, targets, target, a, best, part, kLanes);
}

template <typename T, bool kMask, bool kTop, int kT>
__global__ void __launch_bounds__(kT, (kTop && !kMask ? kResidentTop : kResident) / kT)
    logprob_wide_kernel(Rows r, const T* __restrict__ logits, const uint8_t* __restrict__ masks,
                        const int64_t* __restrict__ targets, Outputs o, int splits, int slots_per_split,
                        Partial* __restrict__ partials, unsigned long long* __restrict__ keys) {
  constexpr int kWarps = kT / kWarp;
  __shared__ Moments sh_m[kWarps];
  __shared__ unsigned long long sh_key[kTop ? kT : 1], sh_cand[kTop ? kCand : 1];
  __shared__ int sh_winner[kTopMax], sh_winners, sh_n;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int64_t row = blockIdx.x / splits;
  const int split = static_cast<int>(blockIdx.x % splits);
  const T* x = logits + row * r.stride;
  const uint8_t* mask = kMask ? masks + row * r.mask_stride : nullptr;
  const RowView<T> view(x, mask, r.width);
  const int lo = split * slots_per_split;
  const int hi = min(lo + slots_per_split, view.slots);
  if (kTop && tid == 0) sh_n = sh_winners = 0;
  Target target{0.0f, 0};
  if (splits > 1) cudaTriggerProgrammaticLaunchCompletion();  // the joining kernel may come and wait
  else target = read_target<T>(r, targets, row, tid, x, mask);

  Moments a;
  const unsigned long long mine = stream_slots<T, kMask, kT>(view, lo, hi, tid, r.c, a);
  const Moments all = block_join<kWarps>(a, r.c, sh_m);

  unsigned long long best = 0;
  if (kTop) {
    // threads whose largest element is among the topk largest such have their elements read again
    const unsigned long long floor = floor_of<kWarps>(mine, r.topk, sh_key);
    const float least = floor ? packed_value(floor) : -kInf;
    const uint32_t least_slot = floor ? packed_rank(floor) : 0xffffffffu;
    if (mine != 0 && mine >= floor) sh_winner[atomicAdd(&sh_winners, 1)] = tid;  // at most topk: keys differ
    __syncthreads();
    const int per = (hi - lo + kT - 1) / kT;  // slots of a thread
    // `use` gets the lanes' keys of one element each, 0 for those that cannot be among the topk
    auto again = [&](auto use) {
      const int pairs = sh_winners * per;
      for (int q = tid; q < ((pairs + kWarp - 1) & -kWarp); q += kT) {
        const int slot = q < pairs ? lo + sh_winner[q / per] + q % per * kT : hi;
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
          use(in ? rank_key(v[i], static_cast<uint32_t>(view.first(slot) + i)) : 0);
        }
      }
    };
    again([&](unsigned long long k) {
      if (k != 0) {
        const int n = atomicAdd(&sh_n, 1);  // any order: they are sorted below
        if (n < kCand) sh_cand[n] = k;
      }
    });
    __syncthreads();
    if (sh_n <= kCand) {
      if (warp == 0) best = merge_list(0, sh_cand, sh_n, lane);
    } else {  // few threads hold many of the largest: merge as they come
      again([&](unsigned long long k) {
        if (__any_sync(kFull, k > __shfl_sync(kFull, best, r.topk - 1)))
          best = merge_best(best, sort_ascending(k, lane), lane);
      });
      sh_key[tid] = best;
      __syncthreads();
      if (warp == 0) best = merge_list(0, sh_key, kT, lane);
    }
  }
  if (splits == 1) {
    finish_row<T>(r, o, row, x, mask, targets, target, all, best, tid, kT);
  } else {
    const int64_t at_split = row * splits + split;
    if (tid == 0) partials[at_split] = {all.m, all.s, all.t, 0.0f};
    if (kTop && tid < r.topk) keys[at_split * r.topk + tid] = best;
  }
}

// One block per row joins its splits, always in the same order.
constexpr int kJoinThreads = 256;
template <typename T, bool kMask>
__global__ void __launch_bounds__(kJoinThreads) logprob_join_kernel(Rows r, const T* __restrict__ logits,
                                                                    const uint8_t* __restrict__ masks,
                                                                    const int64_t* __restrict__ targets, Outputs o,
                                                                    int splits, const Partial* __restrict__ partials,
                                                                    const unsigned long long* __restrict__ keys) {
  constexpr int kWarps = kJoinThreads / kWarp;
  __shared__ Moments sh_m[kWarps];
  __shared__ unsigned long long sh_key[kJoinThreads], sh_cand[kCand];
  __shared__ int sh_n;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int64_t row = blockIdx.x;
  const T* x = logits + row * r.stride;
  const uint8_t* mask = kMask ? masks + row * r.mask_stride : nullptr;
  const Target target = read_target<T>(r, targets, row, tid, x, mask);
  if (tid == 0) sh_n = 0;
  Moments a{-kInf, 0.0f, 0.0f};
  unsigned long long mine = 0, best = 0;
  const unsigned long long* list = keys + row * splits * r.topk;
  cudaGridDependencySynchronize();  // launched while the blocks before it still run
  constexpr int kAhead = 4;
  for (int i = tid; i < splits; i += kJoinThreads * kAhead) {
    Partial p[kAhead];
    unsigned long long k[kAhead];
#pragma unroll
    for (int u = 0; u < kAhead; ++u) {
      const int j = i + u * kJoinThreads;
      p[u] = j < splits ? partials[row * splits + j] : Partial{-kInf, 0.0f, 0.0f, 0.0f};
      k[u] = j < splits && r.topk > 0 ? list[static_cast<int64_t>(j) * r.topk] : 0;  // a split's keys descend
    }
#pragma unroll
    for (int u = 0; u < kAhead; ++u) {
      Moments b{p[u].m, p[u].s, p[u].t};
      const float M = fmaxf(a.m, b.m);
      shift_to(a, M, r.c);
      shift_to(b, M, r.c);
      a = {M, a.s + b.s, a.t + b.t};
      mine = max(mine, k[u]);
    }
  }
  const Moments all = block_join<kWarps>(a, r.c, sh_m);
  if (r.topk > 0) {
    const unsigned long long floor = max(floor_of<kWarps>(mine, r.topk, sh_key), 1ull);
    for (int i = tid; i < splits; i += kJoinThreads)
      for (int q = 0; q < r.topk; ++q) {
        const unsigned long long k = list[static_cast<int64_t>(i) * r.topk + q];
        if (k < floor) break;
        const int n = atomicAdd(&sh_n, 1);
        if (n < kCand) sh_cand[n] = k;
      }
    __syncthreads();
    if (sh_n <= kCand) {
      if (warp == 0) best = merge_list(0, sh_cand, sh_n, lane);
    } else if (warp == 0) {
      const int64_t n = static_cast<int64_t>(splits) * r.topk;
      for (int64_t i = 0; i < n; i += kWarp) {
        const unsigned long long k = i + lane < n ? list[i + lane] : 0;
        if (__any_sync(kFull, k > __shfl_sync(kFull, best, r.topk - 1)))
          best = merge_best(best, sort_ascending(k, lane), lane);
      }
    }
  }
  finish_row<T>(r, o, row, x, mask, targets, target, all, best, tid, kJoinThreads);
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

// dx_j = p_j (a + b log2 p_j) for candidates, with p_j = 2^{y_j} / s and log2 p_j = y_j - log2 s, plus the named
// columns' own gradients / tau.  The row's constants take 1 / s and log2 s in, so that dx_j = 2^{y_j} (a' + b' y_j):
// the exponent carries no rounded log2 s, which would shift every p of a row alike (by 6e-7 at 4.6 M columns).
struct RowGrad {
  float m, a, b;
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
  const float s = u.stats[2 * row + 1];
  const float gh = u.g_entropy ? u.g_entropy[row] : 0.0f;
  const float gl = u.lse ? u.lse[row] : 0.0f;
  const float a = -(named_sum + gh * u.entropy[row] - gl) * r.inv_tau, b = -gh * kLn2 * r.inv_tau;
  g.a = fmaf(-b, log2f(s), a) / s;
  g.b = b / s;
  g.none = s == 0.0f;
  return g;
}

__device__ __forceinline__ float share(const RowGrad& g, float x, float c) {
  const float y = scaled(x, g.m, c);
  return ex2(y) * fmaf(g.b, y, g.a);
}

// The named columns [j_lo, j_hi) once more, with their own gradients added before the one rounding:
// the first to name a column writes it, with all that is named there added in order.
template <typename T, bool kMask, typename Id, typename G>
__device__ __forceinline__ void add_named(const Rows& r, const RowGrad& g, const T* x, const uint8_t* mask, T* grad,
                                          int j_lo, int j_hi, int first, int count, Id id_of, G grad_of) {
  const int n = r.targets + r.topk;
  for (int q = first; q < n; q += count) {
    const int id = id_of(q);
    if (id < j_lo || id >= j_hi || id < 0 || (kMask && mask[id] == 0)) continue;
    float add = 0.0f;
    bool again = false;
    for (int k = 0; k < n; ++k)
      if (id_of(k) == id) {
        again |= k < q;
        add += grad_of(k);
      }
    if (!again) grad[id] = from_f32<T>(fmaf(add, r.inv_tau, share(g, to_f32<T>(x[id]), r.c)));
  }
}

// The gradient of a slot's columns.
template <typename T, bool kMask>
__device__ __forceinline__ void slot_grad(const RowGrad& g, float c, const float (&v)[kVec<T>], T (&out)[kVec<T>]) {
  const Pair m2 = pack2(-g.m, -g.m), c2 = pack2(c, c);
  const Pair a2 = pack2(g.a, g.a), b2 = pack2(g.b, g.b);
#pragma unroll
  for (int i = 0; i < kVec<T>; i += 2) {
    float y0, y1, d0, d1;
    unpack2(mul2(add2(pack2(v[i], v[i + 1]), m2), c2), y0, y1);
    y0 = max_nan(y0, -256.0f);
    y1 = max_nan(y1, -256.0f);
    unpack2(mul2(pack2(ex2(y0), ex2(y1)), fma2(b2, pack2(y0, y1), a2)), d0, d1);
    // a non-candidate reads as -inf: its share is 0 unless the row itself is NaN
    out[i] = from_f32<T>(g.none || (kMask && v[i] == -kInf) ? 0.0f : d0);
    out[i + 1] = from_f32<T>(g.none || (kMask && v[i + 1] == -kInf) ? 0.0f : d1);
  }
}

// The gradient of a thread's slots of [lo, hi), kT apart.
template <typename T, bool kMask, int kT>
__device__ __forceinline__ void slots_grad(const RowView<T>& view, int lo, int hi, int tid, const RowGrad& g, float c,
                                           T* grad) {
  const bool store_vec = (reinterpret_cast<uintptr_t>(grad) - view.lead * sizeof(T)) % 16 == 0;
  auto store = [&](int slot, const T(&out)[kVec<T>], bool whole) {
    const int j0 = view.first(slot);
    if (store_vec && whole) {
      uint4 raw;
      memcpy(&raw, out, 16);
      __stcs(reinterpret_cast<uint4*>(grad + j0), raw);
    } else {
#pragma unroll
      for (int i = 0; i < kVec<T>; ++i)
        if (j0 + i >= 0 && j0 + i < view.width) grad[j0 + i] = out[i];
    }
  };
  for_slots<T, kT>(
      view, lo, hi, tid,
      [&](int slot, int n, auto full) {
        typename RowView<T>::Raw raw[kUnroll];
#pragma unroll
        for (int w = 0; w < kUnroll; ++w)
          if (full || w < n) raw[w] = view.template fetch<kMask>(slot + w * kT);
#pragma unroll
        for (int w = 0; w < kUnroll; ++w) {
          if (!full && w >= n) break;
          float v[kVec<T>];
          T out[kVec<T>];
          view.template values<kMask>(raw[w], v);
          slot_grad<T, kMask>(g, c, v, out);
          store(slot + w * kT, out, true);
        }
      },
      [&](int slot) {
        float v[kVec<T>];
        T out[kVec<T>];
        view.template load<kMask>(slot, v);
        slot_grad<T, kMask>(g, c, v, out);
        store(slot, out, false);
      });
}

// kLanes lanes per row, for narrow rows with few named columns.
constexpr int kNamedNarrow = 64;
template <typename T, bool kMask, int kLanes>
__global__ void __launch_bounds__(kNarrowThreads) logprob_backward_narrow_kernel(Rows r, const T* __restrict__ logits,
                                                                                 const uint8_t* __restrict__ masks,
                                                                                 Upstream u, T* __restrict__ grads) {
  constexpr int kRows = kNarrowThreads / kLanes;
  __shared__ int sh_id[kRows][kNamedNarrow];
  __shared__ float sh_g[kRows][kNamedNarrow];
  const int part = threadIdx.x % kLanes, own = threadIdx.x / kLanes;
  int64_t row = static_cast<int64_t>(blockIdx.x) * kRows + own;
  if (row - (threadIdx.x & 31) / kLanes >= r.rows) return;  // the whole warp is past the end
  const bool valid = row < r.rows;
  row = min(row, r.rows - 1);
  const T* x = logits + row * r.stride;
  const uint8_t* mask = kMask ? masks + row * r.mask_stride : nullptr;
  T* grad = grads + row * r.width;
  float sum = 0.0f;
  for (int q = part; q < r.targets + r.topk; q += kLanes) {
    int64_t id;
    const float g = named(r, u, row, q, id);
    sh_id[own][q] = static_cast<int>(id);
    sh_g[own][q] = g;
    sum += g;
  }
  const RowGrad g = row_grad(r, u, row, lanes_sum<kLanes>(sum));
  const RowView<T> view(x, mask, r.width);
  if (valid) slots_grad<T, kMask, kLanes>(view, 0, view.slots, part, g, r.c, grad);
  __syncwarp();
  if (valid && !g.none)
    add_named<T, kMask>(r, g, x, mask, grad, 0, r.width, part, kLanes, [&](int q) { return sh_id[own][q]; },
                        [&](int q) { return sh_g[own][q]; });
}

template <typename T, bool kMask, int kT>
__global__ void __launch_bounds__(kT, kResident / kT)
    logprob_backward_kernel(Rows r, const T* __restrict__ logits, const uint8_t* __restrict__ masks, Upstream u,
                            T* __restrict__ grads, int splits, int slots_per_split) {
  constexpr int kWarps = kT / kWarp;
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
  for (int q = tid; q < named_n; q += kT) {
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
  slots_grad<T, kMask, kT>(view, lo, hi, tid, g, r.c, grad);
  if (named_n == 0 || g.none || lo >= hi) return;
  __syncthreads();
  add_named<T, kMask>(r, g, x, mask, grad, view.first(lo), view.first(hi), tid, kT, [&](int q) { return sh_id[q]; },
                      [&](int q) { return sh_g[q]; });
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
  MKG_REQUIRE(p->tau >= 0x1p-60 && p->tau <= 0x1p60, "logprob: tau %g outside [2^-60, 2^60]", p->tau);
  MKG_REQUIRE(p->row_stride >= 0 && p->mask_row_stride >= 0, "logprob: negative row stride");
  *r = Rows{p->rows, p->row_stride, p->mask_row_stride, (int)p->width, (int)p->targets, (int)p->topk,
            (float)(1.4426950408889634 / p->tau), (float)(1.0 / p->tau)};
  return MKG_OK;
}

// How rows are dealt to blocks: `splits` pieces of `slots` 16-byte slots per row.
struct Cut {
  int splits, slots, threads;
};
int64_t most_slots(const mkg_logprob_params* p) {  // of a row, wherever it starts
  const int vec = p->dtype == MKG_F32 ? 4 : 8;
  return (p->width + 2 * vec - 2) / vec;
}
Cut in_pieces(int64_t slots, int64_t piece, int threads) {
  const int64_t splits = std::max<int64_t>((slots + piece / 2) / piece, 1);
  int64_t per = (slots + splits - 1) / splits;
  per = (per + threads - 1) / threads * threads;
  return {(int)((slots + per - 1) / per), (int)per, threads};
}
// Pieces, not one share per resident block: SMs differ in speed, and 64 rows of 4,594,485 fp32 logits cut
// into exactly as many blocks as are resident took 249 us forward and 432 us backward, against 211 us
// (5.6 TB/s) and 345 us (6.8 TB/s, reading and writing) in pieces that are handed out as blocks end.
// A piece costs the forward its ordering of alternatives (1,024 slots: 359 us, 8,192: 233 us) and the
// backward its row's constants (256 slots: 642 us).
constexpr int64_t kForwardPiece = 4096, kBackwardPiece = 2048;
Cut forward_cut(const mkg_logprob_params* p) {
  const int64_t slots = most_slots(p);
  // enough rows to go round: they need no joining (5 to 8 us with its launch)
  if (p->rows >= kManyRows) return in_pieces(slots, slots, 128);
  // about one row per SM: larger blocks instead of several and a join (256 x 17,050: 14 us, 30 us)
  if (p->rows >= 128 && p->rows < 512 && slots < 8192) return in_pieces(slots, slots, 512);
  const int64_t even = slots * p->rows / persistent_blocks(4);  // few rows: smaller pieces, to reach every SM
  return in_pieces(slots, std::min(std::max<int64_t>(even, 1024), kForwardPiece), 128);
}
Cut backward_cut(const mkg_logprob_params* p) {
  const int64_t slots = most_slots(p);
  const int64_t even = slots * p->rows / persistent_blocks(8);
  return in_pieces(slots, std::min(std::max<int64_t>(even, 512), kBackwardPiece), 128);
}

template <typename F> int by_type(int32_t dtype, bool mask, F f) {
  switch (dtype) {
    case MKG_F32: return mask ? f((float*)nullptr, std::true_type()) : f((float*)nullptr, std::false_type());
    case MKG_BF16:
      return mask ? f((__nv_bfloat16*)nullptr, std::true_type()) : f((__nv_bfloat16*)nullptr, std::false_type());
    default: return mask ? f((__half*)nullptr, std::true_type()) : f((__half*)nullptr, std::false_type());
  }
}

constexpr int64_t kEightsWide = 512;
template <typename T> bool fits_eights(const Rows& r) {  // 16 values a lane
  return r.topk <= 8 && (r.width + 2 * kVec<T> - 2) / kVec<T> * kVec<T> <= 128;
}
// Whether a warp streams each row.  65,536 rows of 1,645 fp32 logits: 102 us that way and 102 us held in
// registers, but 146 and 261 us with a mask, 161 and 265 us with 8 alternatives, and bf16 96 and 170 us.  20,000
// rows of 7,275: 115 us, and 129 us with a block each (bf16 79 and 127 us); with alternatives topk of the 32 lanes
// are read again, and past about 5 KB of a row that costs more than a block's ordering (8 of fp32: 185 and 148 us,
// of bf16: 121 and 165 us).
bool streams(const Rows& r, int64_t size) {
  const int64_t bytes = r.width * size;
  return r.rows >= kManyRows && r.width > kEightsWide && (r.topk == 0 ? bytes <= 65536 : bytes * r.topk <= 32 * 5120);
}
bool by_lanes(const Rows& r, int64_t size) { return r.width <= kNarrow || streams(r, size); }
// The gradient of a row by a warp: 65,536 rows of 2,500 bf16 logits 127 us, 241 us with a block each; 20,000 of
// 7,275: 102 and 139 us (fp32 187 and 189 us); 8,000 of 16,001 bf16: 86 and 92 us, but of fp32 176 and 159 us.
bool backward_by_lanes(const Rows& r, int64_t size) {
  return r.targets + r.topk <= kNamedNarrow &&
         (r.width <= kNarrow || (r.rows >= kManyRows && r.width * size <= 32768));
}
int64_t size_of(int32_t dtype) { return dtype == MKG_F32 ? 4 : 2; }

template <typename T, bool kMask>
int launch_narrow(const Rows& r, const void* logits, const uint8_t* mask, const int64_t* targets, const Outputs& o,
                  cudaStream_t st) {
  const T* x = static_cast<const T*>(logits);
  const int most = (r.width + 2 * kVec<T> - 2) / kVec<T>;  // slots of a row
  auto launch = [&](auto slots, auto lanes) {
    constexpr int kRows = kNarrowThreads / decltype(lanes)::value;
    logprob_narrow_kernel<T, kMask, decltype(slots)::value, decltype(lanes)::value>
        <<<(unsigned)((r.rows + kRows - 1) / kRows), kNarrowThreads, 0, st>>>(r, x, mask, targets, o);
  };
  using Eight = std::integral_constant<int, 8>;
  using Warp = std::integral_constant<int, kWarp>;
  const int per = (most + kWarp - 1) / kWarp;  // of a lane
  auto stream = [&](auto lanes) {
    constexpr int kRows = kStreamThreads / decltype(lanes)::value;
    logprob_stream_kernel<T, kMask, decltype(lanes)::value>
        <<<(unsigned)((r.rows + kRows - 1) / kRows), kStreamThreads, 0, st>>>(r, x, mask, targets, o);
  };
  const bool many = r.rows >= kManyRows;
  if (many && fits_eights<T>(r)) launch(std::integral_constant<int, 16 / kVec<T>>(), Eight());
  else if (many && r.topk == 0 && r.width <= kEightsWide) stream(Eight());
  else if (streams(r, sizeof(T))) stream(Warp());
  else if (per <= 1) launch(std::integral_constant<int, 1>(), Warp());
  else if (per <= 2) launch(std::integral_constant<int, 2>(), Warp());
  else if (per <= 4) launch(std::integral_constant<int, 4>(), Warp());
  else if (kVec<T> == 8 || per <= 8) launch(std::integral_constant<int, 8>(), Warp());
  else launch(std::integral_constant<int, 64 / kVec<T>>(), Warp());
  MKG_LAUNCHED("logprob_narrow_kernel");
  return MKG_OK;
}

}  // namespace

size_t logprob_workspace_bytes(const mkg_logprob_params* p) {
  Rows r;
  if (check_params(p, &r) != MKG_OK || by_lanes(r, size_of(p->dtype))) return 0;
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
  MKG_REQUIRE(logits && entropy && lse && (p->targets == 0 || (targets && logprobs)) &&
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
    if (by_lanes(r, sizeof(T))) return launch_narrow<T, kMask>(r, logits, mask, targets, o, st);
    const Cut cut = forward_cut(p);
    MKG_REQUIRE(r.rows * cut.splits < (int64_t(1) << 31), "logprob_forward: too many rows");
    Partial* partials = static_cast<Partial*>(ws);
    unsigned long long* keys = reinterpret_cast<unsigned long long*>(partials + (cut.splits > 1 ? r.rows * cut.splits : 0));
    const unsigned grid = (unsigned)(r.rows * cut.splits);
    auto launch = [&](auto top, auto threads) {
      constexpr int kT = decltype(threads)::value;
      logprob_wide_kernel<T, kMask, decltype(top)::value, kT>
          <<<grid, kT, 0, st>>>(r, x, mask, targets, o, cut.splits, cut.slots, partials, keys);
    };
    using Few = std::integral_constant<int, 128>;
    using Many = std::integral_constant<int, 512>;
    if (r.topk > 0) cut.threads == 128 ? launch(std::true_type(), Few()) : launch(std::true_type(), Many());
    else cut.threads == 128 ? launch(std::false_type(), Few()) : launch(std::false_type(), Many());
    MKG_LAUNCHED("logprob_wide_kernel");
    if (cut.splits > 1) {
      cudaLaunchAttribute early;
      early.id = cudaLaunchAttributeProgrammaticStreamSerialization;
      early.val.programmaticStreamSerializationAllowed = 1;
      cudaLaunchConfig_t config = {};
      config.gridDim = dim3((unsigned)r.rows);
      config.blockDim = dim3(kJoinThreads);
      config.stream = st;
      config.attrs = &early;
      config.numAttrs = 1;
      MKG_CUDA(cudaLaunchKernelEx(&config, logprob_join_kernel<T, kMask>, r, x, mask, targets, o, cut.splits,
                                  (const Partial*)partials, (const unsigned long long*)keys));
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
    if (backward_by_lanes(r, sizeof(T))) {
      auto launch = [&](auto lanes) {
        constexpr int kRows = kNarrowThreads / decltype(lanes)::value;
        logprob_backward_narrow_kernel<T, kMask, decltype(lanes)::value>
            <<<(unsigned)((r.rows + kRows - 1) / kRows), kNarrowThreads, 0, st>>>(r, x, mask, u, static_cast<T*>(grad));
      };
      if (r.rows >= kManyRows && r.width <= kEightsWide) launch(std::integral_constant<int, 8>());
      else launch(std::integral_constant<int, kWarp>());
      MKG_LAUNCHED("logprob_backward_narrow_kernel");
      return MKG_OK;
    }
    const Cut cut = backward_cut(p);
    MKG_REQUIRE(r.rows * cut.splits < (int64_t(1) << 31), "logprob_backward: too many rows");
    const size_t sh = (size_t)(r.targets + r.topk) * 8;
    logprob_backward_kernel<T, kMask, 128><<<(unsigned)(r.rows * cut.splits), 128, sh, st>>>(
        r, x, mask, u, static_cast<T*>(grad), cut.splits, cut.slots);
    MKG_LAUNCHED("logprob_backward_kernel");
    return MKG_OK;
  });
}

}  // namespace mkg
