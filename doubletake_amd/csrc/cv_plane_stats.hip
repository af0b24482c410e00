// The plane-sweep volume read as a distribution over depth planes: log probability of a given plane, entropy, normaliser and the
// most probable planes of every pixel; the gradient of the volume for gradients of these; the plane index of a metric depth.
// Formulas and edge cases: include/doubletake_hip.h.
#include "common.hpp"

#include <hip/hip_fp16.h>
#include <hip/hip_bf16.h>
#include <algorithm>
#include <cmath>

namespace dt {

// unsigned division by a launch constant (multiply, add, shift) for numerators below 2^31: the round-up method of Granlund and Montgomery,
// Division by Invariant Integers using Multiplication, 1994
struct Div {
  uint32_t mul, shift;
};
Div make_div(uint32_t d) {
  uint32_t shift = 0;
  while ((1ull << shift) < d) ++shift;
  return {(uint32_t)(((1ull << 32) * ((1ull << shift) - d)) / d + 1), shift};
}
__device__ __forceinline__ uint32_t divide(uint32_t n, Div d) { return (__umulhi(n, d.mul) + n) >> d.shift; }

struct PlaneFwd {
  const void* vol;
  const uint8_t* mask;
  const int64_t* plane;
  const float* planes;
  float *log_prob, *entropy, *log_sum, *top_log_prob;
  int64_t* top_plane;
  float *top_depth, *row_max, *row_log;
  int64_t vs[4], ms[4], ps[4];
  int b, d, h, w, top;
  float scale, outside;
  Div by_hw, by_w;
  uint32_t first;  // pixel the launch begins at (by_range; 0 with 32-bit offsets)
};
DT_ARG_POINTERS(PlaneFwd, offsetof(PlaneFwd, vol), offsetof(PlaneFwd, mask), offsetof(PlaneFwd, plane), offsetof(PlaneFwd, planes),
                offsetof(PlaneFwd, log_prob), offsetof(PlaneFwd, entropy), offsetof(PlaneFwd, log_sum),
                offsetof(PlaneFwd, top_log_prob), offsetof(PlaneFwd, top_plane), offsetof(PlaneFwd, top_depth),
                offsetof(PlaneFwd, row_max), offsetof(PlaneFwd, row_log));

struct PlaneBwd {
  const void* vol;
  const uint8_t* mask;
  const int64_t* plane;
  const float* entropy;
  const int64_t* top_plane;
  const float *row_max, *row_log, *g_log_prob, *g_entropy, *g_log_sum, *g_top;
  void* grad;
  int64_t vs[4], ms[4], gs[4];
  int b, d, h, w, top;
  float scale;
  Div by_hw, by_w;
  uint32_t first;  // as PlaneFwd's
};
DT_ARG_POINTERS(PlaneBwd, offsetof(PlaneBwd, vol), offsetof(PlaneBwd, mask), offsetof(PlaneBwd, plane), offsetof(PlaneBwd, entropy),
                offsetof(PlaneBwd, top_plane), offsetof(PlaneBwd, row_max), offsetof(PlaneBwd, row_log),
                offsetof(PlaneBwd, g_log_prob), offsetof(PlaneBwd, g_entropy), offsetof(PlaneBwd, g_log_sum),
                offsetof(PlaneBwd, g_top), offsetof(PlaneBwd, grad));

struct PlaneNear {
  const float* depth;
  const float* planes;
  int64_t* out;
  int64_t ps[4];
  int b, d, h, w;
  Div by_hw, by_w;
};
DT_ARG_POINTERS(PlaneNear, offsetof(PlaneNear, depth), offsetof(PlaneNear, planes), offsetof(PlaneNear, out));

__device__ __forceinline__ float to_f32(float v) { return v; }
__device__ __forceinline__ float to_f32(__half v) { return __half2float(v); }
__device__ __forceinline__ float to_f32(__hip_bfloat16 v) { return __bfloat162float(v); }
template <typename T>
__device__ __forceinline__ T from_f32(float v);
template <>
__device__ __forceinline__ float from_f32<float>(float v) { return v; }
template <>
__device__ __forceinline__ __half from_f32<__half>(float v) { return __float2half(v); }
template <>
__device__ __forceinline__ __hip_bfloat16 from_f32<__hip_bfloat16>(float v) { return __float2bfloat16(v); }

struct Pixel {
  uint32_t b, y, x, r;  // r: index inside the image
};
__device__ __forceinline__ Pixel pixel_of(uint32_t p, int h, int w, Div by_hw, Div by_w) {
  Pixel q;
  q.b = divide(p, by_hw);
  q.r = p - q.b * ((uint32_t)h * w);
  q.y = divide(q.r, by_w);
  q.x = q.r - q.y * w;
  return q;
}
// elements from the tensor's first pixel to this one.  Off is 32 bits where every byte that a launch touches lies within 4 GB of its
// tensor's first (the low words of the strides are enough then), 64 bits otherwise
template <typename Off>
__device__ __forceinline__ Off offset_of(const int64_t (&s)[4], const Pixel& q) {
  return (Off)q.b * (Off)s[0] + (Off)q.y * (Off)s[2] + (Off)q.x * (Off)s[3];
}

// the pixel this quad of lanes works on
template <typename Off, typename A>
__device__ __forceinline__ uint32_t quad_pixel(const A& a) {
  const uint32_t at = blockIdx.x * 64u + threadIdx.x / 4;
  return sizeof(Off) == 8 ? a.first + at : at;
}

// A launch-uniform 64-bit base plus an offset in bytes per lane.  The empty statement keeps the base in scalar registers: left to itself
// the compiler adds the two first, a 64-bit vector addition and two registers per access, and hoists the sums out of the loop over
// planes.  Planes innermost, D = 64, 4 alternatives, 8 x 120 x 160 pixels: 60 -> 56 registers and 13.6 -> 13.4 us, with a mask per plane
// 83 -> 66 and 15.9 -> 15.7.  (Not where a lane steps over planes, the hoisted addresses win there: 128 planes of float16, 8 x 240 x 320
// pixels 36.3 us, kept in scalar registers 39.0.)
#define DT_GLOBAL __attribute__((address_space(1)))
template <typename T, typename Off>
__device__ __forceinline__ T load(const void* base, Off off) {
  uint64_t address = (uint64_t)base;
  if constexpr (sizeof(Off) == 4) asm("" : "+s"(address));
  return *(const T*)(const DT_GLOBAL char*)(address + off);
}
template <typename T, typename Off>
__device__ __forceinline__ void store(void* base, Off off, T v) {
  uint64_t address = (uint64_t)base;
  if constexpr (sizeof(Off) == 4) asm("" : "+s"(address));
  *(T*)(DT_GLOBAL char*)(address + off) = v;
}

// scale (x - m) - ls for the outputs: halves, so that two scores at opposite ends of the float range do not overflow in between
__device__ __forceinline__ float log_prob_of(float x, float m, float ls, float scale) {
  return 2.f * ((0.5f * x - 0.5f * m) * scale) - ls;
}

// ---- alternatives ------------------------------------------------------------------------------------------------------------
// A score and its plane as ONE double, so that a compare-exchange of the ordered lists is one v_max_f64 and one v_min_f64: the
// float's bits are the high word, which orders sign and magnitude like the float itself (its 8 exponent bits and 3 mantissa bits
// become the double's 11 exponent bits; +-inf gives 0x7f8, so no score becomes a double NaN), and the plane is the low word,
// complemented for positive scores: of equal scores the lower plane is the larger double.  -0 counts as +0; every NaN becomes
// 0x7fe00000, above +inf.
constexpr uint32_t kNone = 0xff800000u;  // -inf: a masked plane, an empty slot
__device__ __forceinline__ double make_key(uint32_t hi, uint32_t lo) { return __longlong_as_double((long long)((uint64_t)hi << 32 | lo)); }
__device__ __forceinline__ double key_of(float x, int plane) {
  const float c = x + 0.f;
  const uint32_t hi = c != c ? 0x7fe00000u : __float_as_uint(c);
  return make_key(hi, ~(uint32_t)plane ^ (uint32_t)((int32_t)hi >> 31));
}
__device__ __forceinline__ uint32_t key_hi(double k) { return (uint32_t)((uint64_t)__double_as_longlong(k) >> 32); }
__device__ __forceinline__ int key_plane(double k) {
  return (int)~((uint32_t)__double_as_longlong(k) ^ (uint32_t)((int32_t)key_hi(k) >> 31));
}
// the same score, `by` planes further on
__device__ __forceinline__ double key_moved(double k, int by) {
  const uint32_t hi = key_hi(k), sign = (uint32_t)((int32_t)hi >> 31);
  return make_key(hi, (uint32_t)__double_as_longlong(k) - (((uint32_t)by ^ sign) - sign));
}
__device__ __forceinline__ void order(double& a, double& b) {
  const double hi = fmax(a, b), lo = fmin(a, b);
  a = hi, b = lo;
}
// descending sort of K keys (the smallest networks: 1, 5 and 19 exchanges)
template <int K>
__device__ __forceinline__ void sort_keys(double (&k)[K]) {
  if constexpr (K == 4) {
    order(k[0], k[2]), order(k[1], k[3]);
    order(k[0], k[1]), order(k[2], k[3]);
    order(k[1], k[2]);
  } else if constexpr (K == 8) {
    order(k[0], k[2]), order(k[1], k[3]), order(k[4], k[6]), order(k[5], k[7]);
    order(k[0], k[4]), order(k[1], k[5]), order(k[2], k[6]), order(k[3], k[7]);
    order(k[0], k[1]), order(k[2], k[3]), order(k[4], k[5]), order(k[6], k[7]);
    order(k[2], k[4]), order(k[3], k[5]);
    order(k[1], k[4]), order(k[3], k[6]);
    order(k[1], k[2]), order(k[3], k[4]), order(k[5], k[6]);
  }
}
// the K largest of two descending lists: the element-wise maxima of one against the other reversed are those K, and a bitonic
// sequence, which log2 K rounds of exchanges put in order
template <int K>
__device__ __forceinline__ void merge_keys(double (&k)[K], const double (&o)[K]) {
#pragma unroll
  for (int i = 0; i < K; ++i) k[i] = fmax(k[i], o[K - 1 - i]);
#pragma unroll
  for (int dist = K / 2; dist > 0; dist /= 2)
#pragma unroll
    for (int i = 0; i < K; ++i)
      if (!(i & dist)) order(k[i], k[i + dist]);
}

// ---- exchange inside groups of G = 1, 4 neighbouring lanes ---------------------------------------------------------------------------
template <int STEP>
__device__ __forceinline__ uint32_t other_u32(uint32_t v) {  // lane ^ STEP
  constexpr int ctrl = STEP == 1 ? 0xB1 : 0x4E;  // quad_perm 1,0,3,2 / 2,3,0,1
  return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, ctrl, 0xf, 0xf, true);
}
template <int STEP>
__device__ __forceinline__ float other(float v) { return __uint_as_float(other_u32<STEP>(__float_as_uint(v))); }
template <int STEP>
__device__ __forceinline__ double other(double v) {
  const uint64_t b = (uint64_t)__double_as_longlong(v);
  return make_key(other_u32<STEP>((uint32_t)(b >> 32)), other_u32<STEP>((uint32_t)b));
}
template <int G>
__device__ __forceinline__ float group_max(float v) {
  if constexpr (G == 4) v = fmaxf(v, other<1>(v)), v = fmaxf(v, other<2>(v));
  return v;
}
template <int G>
__device__ __forceinline__ float group_sum(float v) {
  if constexpr (G == 4) v += other<1>(v), v += other<2>(v);
  return v;
}
template <int K, int STEP>
__device__ __forceinline__ void merge_lanes(double (&k)[K]) {
  double o[K];
#pragma unroll
  for (int j = 0; j < K; ++j) o[j] = other<STEP>(k[j]);
  merge_keys(k, o);
}

// ---- running statistics of one lane --------------------------------------------------------------------------------------------
// m: largest score so far (-inf: none); with y = c (x - m), c = scale log2 e: s = sum 2^y and t = sum 2^y y.  When the maximum moves
// by delta = c (m_old - m_new): s' = s 2^delta, t' = (t + delta s) 2^delta.  A NaN score, or +inf (inf - inf), makes s and with it
// every statistic NaN; the clamp keeps 0 * -inf out of t.  Differences come before the product: scores far from zero lose nothing.
// s and t are float32: at D planes a lane adds D / 16 partial sums to them and moves its maximum D / 16 times at most, 4 roundings of 2^-24
// each, so that ln s is off by D / 4 + 6 ln D + 40 of them at worst: DT_PLANE_MAX_PLANES keeps that below 1e-3 (64 planes: 5e-6).
// The G lanes of a group that share a pixel move their maximum together, so that their sums need no rescaling when they join.
constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;
template <int K>
struct Stats {
  float m = -INFINITY, s = 0.f, t = 0.f;
  double key[K > 0 ? K : 1];
  __device__ __forceinline__ Stats() {
#pragma unroll
    for (int j = 0; j < K; ++j) key[j] = make_key(kNone, 0xffffffffu);
  }
  __device__ __forceinline__ void rebase(float to, float c) {
    if (s != 0.f) {  // (nothing to move, and -inf - -inf, otherwise)
      const float delta = fmaxf(c * (m - to), -1e4f);
      const float r = __builtin_amdgcn_exp2f(delta);
      t = (t + delta * s) * r;
      s *= r;
    }
    m = to;
  }
  // N more scores (masked ones are -inf), of planes plane(0) < plane(1) < ...
  template <int G, int N, typename F>
  __device__ __forceinline__ void add(const float (&x)[N], float c, F plane) {
    float top = m;
#pragma unroll
    for (int e = 0; e < N; ++e) top = fmaxf(top, x[e]);
    top = group_max<G>(top);
    if (top != m) rebase(top, c);
    const float m0 = m == -INFINITY ? 0.f : m;
    float ps = 0.f, pt = 0.f;  // (of these N alone: s and t round once per N planes, not once per plane)
#pragma unroll
    for (int e = 0; e < N; ++e) {
      const float y = c * (x[e] - m0);
      const float ex = __builtin_amdgcn_exp2f(y);
      ps += ex;
      pt += ex * fmaxf(y, -1e4f);
    }
    s += ps, t += pt;
    if constexpr (K > 0) {
      static_assert(N % K == 0);
#pragma unroll
      for (int b = 0; b < N; b += K) {
        double k[K];
#pragma unroll
        for (int j = 0; j < K; ++j) k[j] = key_of(x[b + j], plane(b + j));
        sort_keys(k);
        merge_keys(key, k);
      }
    }
  }
};

// Writes a pixel's outputs from its statistics, which G lanes hold alike: lane 0 the real values, lane j the alternatives j, j + G, ...
template <int K, int G, typename Off>
__device__ __forceinline__ void write(const PlaneFwd& a, uint32_t p, const Pixel& q, const Stats<K>& st, int64_t given, float x_given, int lane) {
  const float s = st.s, t = st.t;
  const float m = st.m == -INFINITY ? 0.f : st.m;
  const bool empty = s == 0.f;
  const float ls = kLn2 * __builtin_amdgcn_logf(s);  // (s is 0, NaN or at least 1)
  const Off po = (Off)p * 4;
  if (lane == 0) {
    store(a.entropy, po, empty ? 0.f : ls - kLn2 * (t * __builtin_amdgcn_rcpf(s)));
    store(a.log_sum, po, m * a.scale + ls);
    if (a.row_max) store(a.row_max, po, m), store(a.row_log, po, ls);
    if (a.plane) store(a.log_prob, po, given < 0 || given >= a.d ? a.outside : empty ? -INFINITY : log_prob_of(x_given, m, ls, a.scale));
  }
  if constexpr (K > 0) {
    const Off hw = (Off)a.h * a.w;
    Off o = ((Off)q.b * a.top + lane) * hw + q.r;
#pragma unroll
    for (int j = 0; j < K; j += G, o += G * hw) {
      double k = st.key[j];
#pragma unroll
      for (int i = 1; i < G && j + i < K; ++i) {
        const double other_slot = st.key[j + i];  // (read before it is chosen: a chosen read would move the list to memory)
        k = lane == i ? other_slot : k;
      }
      if (j + lane >= a.top) break;
      const bool none = key_hi(k) == kNone;
      const int at = key_plane(k);
      store<int64_t>(a.top_plane, o * 8, none ? -1 : at);
      store(a.top_log_prob, o * 4, none ? -INFINITY : log_prob_of(__uint_as_float(key_hi(k)), m, ls, a.scale));
      if (a.top_depth) {
        const float depth = none ? 0.f : load<float>(a.planes, (Off)((offset_of<Off>(a.ps, q) + (Off)at * (Off)a.ps[1]) * 4));
        store(a.top_depth, o * 4, depth);
      }
    }
  }
}

// ---- reading scores ----------------------------------------------------------------------------------------------------------------
// A mask that does not vary over the planes is read once per pixel by the kernels; the readers apply one that does.

// the score of one plane of a pixel, -inf where the mask hides it
template <typename T, typename Off>
__device__ __forceinline__ float score_first(const PlaneFwd& a, Off vo, Off mo, int64_t d) {
  const bool seen = !a.mask || a.mask[d * a.ms[1] + mo];
  return seen ? to_f32(*(const T*)((const char*)a.vol + d * a.vs[1] * (int64_t)sizeof(T) + vo)) : -INFINITY;
}

template <typename T, typename Off>
__device__ __forceinline__ float score_last(const PlaneFwd& a, Off vo, Off mo, int d) {
  const bool seen = !a.mask || load<uint8_t>(a.mask, (Off)(mo + (Off)d * (Off)a.ms[1]));
  return seen ? to_f32(load<T>(a.vol, (Off)(vo + (Off)d * (Off)sizeof(T)))) : -INFINITY;
}

struct __attribute__((packed)) Packed4 {
  uint32_t bytes;
};
template <typename T, int N>
struct Vec {  // aligned like one element: global memory accesses need no more
  T v[N];
};
// N planes' scores and mask bytes as they come from memory.  Loading and unpacking are apart so that other work goes in between.
template <typename T, int N>
struct Raw {
  T v[N];
  uint8_t seen[N];
  uint32_t word[N / 4];
};

// N planes d0, d0 + 1, ... of one pixel; those from `end` on count as -inf.  All loads are in flight together and none is guarded
// (past the end the last plane is read again): a guard per load makes the compiler wait for each.
template <typename T, int N, typename Off, typename A>
__device__ __forceinline__ void load_first(Raw<T, N>& raw, const A& a, bool masked, int d0, int end, Off vo, Off mo) {
  const char* vol = (const char*)a.vol + vo;
  const uint8_t* mask = a.mask + mo;
#pragma unroll
  for (int e = 0; e < N; ++e) raw.v[e] = ((const T*)vol)[min(d0 + e, end - 1) * a.vs[1]];
  if (masked) {
#pragma unroll
    for (int e = 0; e < N; ++e) raw.seen[e] = mask[min(d0 + e, end - 1) * a.ms[1]];
  }
}
template <typename T, int N>
__device__ __forceinline__ void unpack_first(float (&x)[N], const Raw<T, N>& raw, bool masked, int d0, int end) {
  if (masked) {
#pragma unroll
    for (int e = 0; e < N; ++e) x[e] = raw.seen[e] ? to_f32(raw.v[e]) : -INFINITY;
  } else {
#pragma unroll
    for (int e = 0; e < N; ++e) x[e] = to_f32(raw.v[e]);
  }
  if (d0 + N > end) {
#pragma unroll
    for (int e = 0; e < N; ++e) x[e] = d0 + e < end ? x[e] : -INFINITY;
  }
}

// Layout of N planes per lane among G lanes of a pixel, from plane d0 on, 16 bytes per lane and load: plane of element e of lane 0; lane
// l's is l * kVec further on
template <typename T, int G>
struct Spread {
  static constexpr int kVec = 16 / sizeof(T), kStep = G * kVec;
  __device__ __forceinline__ static int plane(int d0, int e) { return d0 + (e / kVec) * kStep + e % kVec; }
};
// What the readers below know about the mask at compile time: none that varies over the planes, one byte per load, or the planes' bytes
// next to each other like the scores (a comparison of a channels_last volume): then as many bytes per load as scores, taken apart when
// they are used.  (One kernel for all three would hold the addresses and branches of each.)
enum MaskKind { kNoMask, kMaskBytes, kMaskVectors };
template <MaskKind M, typename T, int G, int N, typename Off, typename A>
__device__ __forceinline__ void load_last(Raw<T, N>& raw, const A& a, int d0, int lane, Off vo, Off mo) {
  using L = Spread<T, G>;
  constexpr int kVec = L::kVec;
  const Off lvo = vo + lane * 16u, lmo = mo + (Off)(lane * kVec) * (Off)a.ms[1];
  if (d0 + N * G <= a.d) {
#pragma unroll
    for (int e = 0; e < N; e += kVec) {
      const Vec<T, kVec> v = load<Vec<T, kVec>>((const T*)a.vol + L::plane(d0, e), lvo);
#pragma unroll
      for (int j = 0; j < kVec; ++j) raw.v[e + j] = v.v[j];
    }
    if constexpr (M == kMaskVectors) {
#pragma unroll
      for (int e = 0; e < N; e += kVec) {
        const Vec<Packed4, kVec / 4> v = load<Vec<Packed4, kVec / 4>>(a.mask + L::plane(d0, e), lmo);
#pragma unroll
        for (int j = 0; j < kVec / 4; ++j) raw.word[e / 4 + j] = v.v[j].bytes;
      }
    } else if constexpr (M == kMaskBytes) {
#pragma unroll
      for (int e = 0; e < N; ++e) raw.seen[e] = load<uint8_t>(a.mask + L::plane(d0, e) * a.ms[1], lmo);
    }
  } else {
#pragma unroll
    for (int e = 0; e < N; e += kVec) {
      const int left = a.d - L::plane(d0, e) - lane * kVec;  // planes from this lane's first on
#pragma unroll
      for (int j = 0; j < kVec; ++j) raw.v[e + j] = T(), raw.seen[e + j] = 0;
      if (L::plane(d0, e) + L::kStep <= a.d) {
        const Vec<T, kVec> v = load<Vec<T, kVec>>((const T*)a.vol + L::plane(d0, e), lvo);
#pragma unroll
        for (int j = 0; j < kVec; ++j) raw.v[e + j] = v.v[j];
      } else if (left > 0) {
#pragma unroll
        for (int j = 0; j < kVec; ++j)
          raw.v[e + j] = load<T>((const T*)a.vol + L::plane(d0, e), (Off)(lvo + (Off)min(j, left - 1) * (Off)sizeof(T)));
      }
      if (M != kNoMask && left > 0) {
#pragma unroll
        for (int j = 0; j < kVec; ++j)
          raw.seen[e + j] = load<uint8_t>(a.mask + L::plane(d0, e) * a.ms[1], (Off)(lmo + (Off)min(j, left - 1) * (Off)a.ms[1]));
      }
    }
  }
}
template <MaskKind M, typename T, int G, int N>
__device__ __forceinline__ void unpack_last(float (&x)[N], const Raw<T, N>& raw, int d0, int planes, int lane) {
  using L = Spread<T, G>;
  if (d0 + N * G <= planes) {
#pragma unroll
    for (int e = 0; e < N; ++e) {
      const bool seen = M == kNoMask || (M == kMaskVectors ? (raw.word[e / 4] & (0xffu << e % 4 * 8)) != 0 : raw.seen[e] != 0);
      x[e] = seen ? to_f32(raw.v[e]) : -INFINITY;
    }
  } else {
#pragma unroll
    for (int e = 0; e < N; ++e)
      x[e] = L::plane(d0, e) + lane * L::kVec < planes && (M == kNoMask || raw.seen[e]) ? to_f32(raw.v[e]) : -INFINITY;
  }
}

// ---- statistics --------------------------------------------------------------------------------------------------------------------
constexpr int kN = 16;  // planes per lane in registers

// the first half of a lane's planes, where the second lies past the end
template <int G, int K, typename F>
__device__ __forceinline__ void add_planes(Stats<K>& st, const float (&x)[kN], float c, bool half, F plane) {
  if (half) {
    float y[kN / 2];
#pragma unroll
    for (int e = 0; e < kN / 2; ++e) y[e] = x[e];
    st.template add<G>(y, c, plane);
  } else {
    st.template add<G>(x, c, plane);
  }
}

// Volume with neighbouring pixels next to each other (NCHW; any strides work): one lane per pixel.
// S = 4: the four waves of a workgroup share 64 pixels, a quarter of the planes each; the partial results change places through LDS so
// that four neighbouring lanes hold the four parts of a pixel, and all waves join and write 16 pixels each.
// Bound: memory in float32 (16 x 64 x 120 x 160 pixels, 4 alternatives: 21.2 us, 4.7 TB/s of what has to move; a large copy on this card
// reaches 4.8) and in float16 without alternatives (8 x 128 x 240 x 320: 36.3 us, 4.7 TB/s).  In float16 with alternatives (16 x 64 x 120
// x 160, 4 of them: 20.0 us, 3.0 TB/s) memory (12.5 us) and vector instructions (1538 a wave, 12.5 us) take turns: a lane has nothing in
// flight during its arithmetic, and 4.7 waves per SIMD cover a part.  Latency below about 50000 pixels (one keyframe 4.2 to 5.3 us).
template <typename T, int K, int S, typename Off>
__global__ void __launch_bounds__(256) plane_stats_first_kernel(PlaneFwd a) {
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64), lane = threadIdx.x % 64;
  const uint32_t pixels = (uint32_t)a.b * a.h * a.w, first = blockIdx.x * (256u / S);
  const float c = a.scale * kLog2e;
  // the pixel this lane writes (and, S == 1, the one it reads)
  const uint32_t at = first + threadIdx.x / S, p = min(at, pixels - 1);
  const int group = threadIdx.x % S;
  const Pixel q = pixel_of(p, a.h, a.w, a.by_hw, a.by_w);
  const Off mo = offset_of<Off>(a.ms, q), vo = offset_of<Off>(a.vs, q) * (Off)sizeof(T);
  const bool masked = a.mask && a.ms[1] != 0;
  const uint8_t seen = a.mask && !masked ? load<uint8_t>(a.mask, mo) : 1;  // (used after the loop: nothing waits for it here)
  const int64_t given = a.plane ? load<int64_t>(a.plane, (Off)p * 8) : -1;
  Off rvo = vo, rmo = mo;
  int begin = 0, end = a.d;
  if constexpr (S > 1) {
    const Pixel r = pixel_of(min(first + lane, pixels - 1), a.h, a.w, a.by_hw, a.by_w);
    rvo = offset_of<Off>(a.vs, r) * (Off)sizeof(T), rmo = offset_of<Off>(a.ms, r);
    const int part = (a.d + S - 1) / S;
    begin = wave * part, end = min(a.d, begin + part);
  }
  Stats<K> st;
  for (int d0 = begin; d0 < end; d0 += kN) {
    Raw<T, kN> raw;
    load_first(raw, a, masked, d0, end, rvo, rmo);
    float x[kN];
    unpack_first(x, raw, masked, d0, end);
    add_planes<1>(st, x, c, d0 + kN / 2 >= end, [&](int e) { return d0 + e; });
  }
  if constexpr (S > 1) {
    constexpr int kRow = 64 + 16;  // (the four parts of 16 pixels fall into different banks)
    __shared__ float part_f[3][S * kRow];
    __shared__ double part_k[K > 0 ? K : 1][S * kRow];
    const int put = wave * kRow + lane;
    part_f[0][put] = st.m, part_f[1][put] = st.s, part_f[2][put] = st.t;
#pragma unroll
    for (int j = 0; j < K; ++j) part_k[j][put] = st.key[j];
    __syncthreads();
    const int get = group * kRow + threadIdx.x / S;
    st.m = part_f[0][get], st.s = part_f[1][get], st.t = part_f[2][get];
#pragma unroll
    for (int j = 0; j < K; ++j) st.key[j] = part_k[j][get];
    const float top = group_max<S>(st.m);
    if (top != st.m) st.rebase(top, c);
    st.s = group_sum<S>(st.s), st.t = group_sum<S>(st.t);
    if constexpr (K > 0) merge_lanes<K, 1>(st.key), merge_lanes<K, 2>(st.key);
  }
  if (!seen) st = Stats<K>();
  const float x_given = group == 0 && given >= 0 && given < a.d ? score_first<T>(a, vo, mo, given) : 0.f;
  if (at < pixels) write<K, S, Off>(a, p, q, st, given, x_given, group);
}

// Volume with the planes of a pixel next to each other (channels_last): four lanes per pixel, 8 planes per lane at a time.  Two loads of
// a lane cover the halves of a 128-byte line, so four lanes fetch whole lines; 16 lanes per pixel would pay more for joining and writing.
// Bound: memory from about 64 float32 planes on (16 x 64 x 120 x 160, 4 alternatives: 21.2 us, 4.7 TB/s).  Below, memory and the vector
// instructions of joining and writing a pixel together (8 x 32 x 120 x 160: 9.9 us, memory 6.2, 350 instructions a wave 5.6); in float16
// vector instructions (16 x 64 x 120 x 160: 21.3 us, 535 a wave 17.3, memory 12.5); latency at one keyframe (3.6 to 4.8 us).
template <typename T, int K, MaskKind M, typename Off>
__global__ void __launch_bounds__(256) plane_stats_last_kernel(PlaneFwd a) {
  constexpr int G = 4, N = 8;
  using L = Spread<T, G>;
  const int lane = threadIdx.x % G;
  const uint32_t at = quad_pixel<Off>(a);
  const uint32_t pixels = (uint32_t)a.b * a.h * a.w;
  const uint32_t p = min(at, pixels - 1);
  const Pixel q = pixel_of(p, a.h, a.w, a.by_hw, a.by_w);
  const Off vo = offset_of<Off>(a.vs, q) * (Off)sizeof(T), mo = offset_of<Off>(a.ms, q);
  const float c = a.scale * kLog2e;
  const uint8_t seen = M == kNoMask && a.mask ? load<uint8_t>(a.mask, mo) : 1;  // (used after the loop: nothing waits for it here)
  const int64_t given = a.plane ? load<int64_t>(a.plane, (Off)p * 8) : -1;
  Stats<K> st;
  Raw<T, N> raw;
  load_last<M, T, G>(raw, a, 0, lane, vo, mo);
  for (int d0 = 0; d0 < a.d; d0 += N * G) {
    float x[N];
    unpack_last<M, T, G>(x, raw, d0, a.d, lane);
    if (d0 + N * G < a.d) load_last<M, T, G>(raw, a, d0 + N * G, lane, vo, mo);  // (under way during the arithmetic)
    st.template add<G>(x, c, [&](int e) { return L::plane(d0, e); });
  }
  st.s = group_sum<G>(st.s), st.t = group_sum<G>(st.t);
  if constexpr (K > 0) {
#pragma unroll
    for (int j = 0; j < K; ++j) st.key[j] = key_moved(st.key[j], lane * L::kVec);
    merge_lanes<K, 1>(st.key), merge_lanes<K, 2>(st.key);
  }
  if (!seen) st = Stats<K>();
  const float x_given = lane == 0 && given >= 0 && given < a.d ? score_last<T>(a, vo, mo, (int)given) : 0.f;
  if (at < pixels) write<K, G, Off>(a, p, q, st, given, x_given, lane);
}

// ---- gradient ------------------------------------------------------------------------------------------------------------------
// What a pixel contributes to each of its planes: with l = c (x - m) - log2 s the plane's log probability in base 2,
//   dx = 2^l (k0 + k1 max(l, -1e4)) + (gradient of the slot that names the plane),
//   k0 = scale (g_log_sum - g_log_prob - sum g_top - g_entropy entropy), k1 = -scale g_entropy ln 2.
// Slots: the alternatives and the given plane, which is folded into the alternative it coincides with; all planes differ.
template <int K, typename Off>
struct Pull {
  float m, ls2, c, k0, k1;
  bool hidden;
  int at[K + 1];
  float g[K + 1];
  __device__ __forceinline__ Pull(const PlaneBwd& a, uint32_t p, const Pixel& q, bool hidden) : hidden(hidden) {
    // (loads first, none behind a condition on another's value)
    const Off po = (Off)p * 4;
    m = load<float>(a.row_max, po);
    const float ls = load<float>(a.row_log, po), ent = load<float>(a.entropy, po);
    const float ge = a.g_entropy ? load<float>(a.g_entropy, po) : 0.f;
    float all = a.g_log_sum ? load<float>(a.g_log_sum, po) : 0.f;
    const int64_t given = a.g_log_prob ? load<int64_t>(a.plane, po * 2) : -1;
    g[K] = a.g_log_prob ? load<float>(a.g_log_prob, po) : 0.f;
    const Off hw = (Off)a.h * a.w, o = (Off)q.b * a.top * hw + q.r;
#pragma unroll
    for (int j = 0; j < K; ++j) {
      at[j] = j < a.top ? (int)load<int64_t>(a.top_plane, (Off)((o + j * hw) * 8)) : -1;
      g[j] = j < a.top ? load<float>(a.g_top, (Off)((o + j * hw) * 4)) : 0.f;
    }
    const bool inside = given >= 0 && given < a.d;
    at[K] = inside ? (int)given : -1, g[K] = inside ? g[K] : 0.f;
    all -= g[K];
#pragma unroll
    for (int j = 0; j < K; ++j) {
      g[j] = at[j] < 0 ? 0.f : g[j];
      all -= g[j];
      const bool same = at[j] >= 0 && at[j] == at[K];
      g[j] = a.scale * (same ? g[j] + g[K] : g[j]);
      at[K] = same ? -1 : at[K];
    }
    g[K] *= a.scale;
    ls2 = ls * kLog2e, c = a.scale * kLog2e;
    k0 = a.scale * (ge != 0.f ? all - ge * ent : all);
    k1 = -a.scale * kLn2 * ge;
  }
  // d: the plane, x: its score, -inf where the mask hides it
  __device__ __forceinline__ float operator()(int d, float x) const {
    const float l = c * (x - m) - ls2;
    float slot = 0.f;
#pragma unroll
    for (int j = 0; j <= K; ++j) slot = d == at[j] ? g[j] : slot;
    const float v = __builtin_amdgcn_exp2f(l) * (k0 + k1 * fmaxf(l, -1e4f)) + slot;
    return hidden || x == -INFINITY ? 0.f : v;
  }
  // number the planes from another one
  __device__ __forceinline__ void move(int by) {
#pragma unroll
    for (int j = 0; j <= K; ++j) at[j] = at[j] < 0 ? INT32_MIN : at[j] + by;
  }
};

// neighbouring pixels next to each other: one lane per pixel and 16 planes, blockIdx.y numbers the groups of planes
// Bound: memory (float16, 16 x 64 x 96 x 128: 13.0 us, 4.3 TB/s of what has to move; the pixels' statistics are read once per 16 planes)
template <typename T, int K, typename Off>
__global__ void __launch_bounds__(256) plane_grad_first_kernel(PlaneBwd a) {
  const uint32_t p = blockIdx.x * 256u + threadIdx.x;
  if (p >= (uint32_t)a.b * a.h * a.w) return;
  const Pixel q = pixel_of(p, a.h, a.w, a.by_hw, a.by_w);
  const Off vo = offset_of<Off>(a.vs, q) * (Off)sizeof(T), mo = offset_of<Off>(a.ms, q), go = offset_of<Off>(a.gs, q) * (Off)sizeof(T);
  const bool masked = a.mask && a.ms[1] != 0;
  for (int d0 = blockIdx.y * kN; d0 < a.d; d0 += gridDim.y * kN) {
    Raw<T, kN> raw;
    load_first(raw, a, masked, d0, a.d, vo, mo);
    const Pull<K, Off> pull(a, p, q, a.mask && !masked && !load<uint8_t>(a.mask, mo));
    float x[kN];
    unpack_first(x, raw, masked, d0, a.d);
    T* grad = (T*)((char*)a.grad + go);
#pragma unroll
    for (int e = 0; e < kN; ++e) {
      if (d0 + e >= a.d) break;
      grad[(d0 + e) * a.gs[1]] = from_f32<T>(pull(d0 + e, x[e]));
    }
  }
}

// the planes of a pixel next to each other, in the volume and in its gradient: four lanes per pixel, 16 bytes per lane, load and store
// Bound: memory (4 x 256 x 120 x 160, mask, 4 alternatives: 37.7 us, 4.8 TB/s)
template <typename T, int K, MaskKind M, typename Off>
__global__ void __launch_bounds__(256) plane_grad_last_kernel(PlaneBwd a) {
  constexpr int G = 4, N = 8;
  using L = Spread<T, G>;
  const int lane = threadIdx.x % G;
  const uint32_t p = quad_pixel<Off>(a);
  if (p >= (uint32_t)a.b * a.h * a.w) return;
  const Pixel q = pixel_of(p, a.h, a.w, a.by_hw, a.by_w);
  const Off vo = offset_of<Off>(a.vs, q) * (Off)sizeof(T), mo = offset_of<Off>(a.ms, q), go = offset_of<Off>(a.gs, q) * (Off)sizeof(T);
  Raw<T, N> raw;
  load_last<M, T, G>(raw, a, 0, lane, vo, mo);
  Pull<K, Off> pull(a, p, q, M == kNoMask && a.mask && !load<uint8_t>(a.mask, mo));
  pull.move(-lane * L::kVec);
  for (int d0 = 0;;) {
    float x[N];
    unpack_last<M, T, G>(x, raw, d0, a.d, lane);
#pragma unroll
    for (int e = 0; e < N; e += L::kVec) {
      const int d = L::plane(d0, e) + lane * L::kVec;
      Vec<T, L::kVec> r;
#pragma unroll
      for (int j = 0; j < L::kVec; ++j) r.v[j] = from_f32<T>(pull(L::plane(d0, e + j), x[e + j]));
      if (d + L::kVec <= a.d) {
        store((T*)a.grad + L::plane(d0, e), (Off)(go + lane * 16u), r);
      } else {
#pragma unroll
        for (int j = 0; j < L::kVec; ++j)
          if (d + j < a.d) store((T*)a.grad + L::plane(d0, e) + j, (Off)(go + lane * 16u), r.v[j]);
      }
    }
    d0 += N * G;
    if (d0 >= a.d) break;
    load_last<M, T, G>(raw, a, d0, lane, vo, mo);
  }
}

// ---- planes of depths ------------------------------------------------------------------------------------------------------------
// 64-bit differences of 32-bit depths are exact within a factor of 2^29 (24 + 29 = 53 bits), so a tie is a tie there; beyond, rounding keeps
// the order of the differences but may make equal ones of them.  16 planes' loads are in flight together.
// Workgroups of one wave: a keyframe's 300 waves spread over all compute units (19200 pixels, 64 planes: 4.7 us, 5.1 with four waves).
// Bound: memory where planes vary over the image (8 x 96 x 240 x 320: 46.7 us, 5.2 TB/s, a part from the last-level cache; with four waves
// 44.3), else latency.
__global__ void __launch_bounds__(64) nearest_planes_kernel(PlaneNear a) {
  const uint32_t p = blockIdx.x * 64u + threadIdx.x;
  if (p >= (uint32_t)a.b * a.h * a.w) return;
  const Pixel q = pixel_of(p, a.h, a.w, a.by_hw, a.by_w);
  const float* planes = a.planes + offset_of<int64_t>(a.ps, q);
  const float depth = a.depth[p];
  int at = -1;
  double best = INFINITY;
  for (int d0 = 0; d0 < a.d; d0 += kN) {
    float v[kN];
#pragma unroll
    for (int e = 0; e < kN; ++e) v[e] = planes[min(d0 + e, a.d - 1) * a.ps[1]];  // (the last plane again: never nearer than itself)
#pragma unroll
    for (int e = 0; e < kN; ++e) {
      const double off = fabs((double)v[e] - (double)depth);
      if (off < best) best = off, at = d0 + e;
    }
  }
  a.out[p] = depth > 0.f && depth < INFINITY ? at : -1;
}

template <typename F>
void by_type(int dtype, F&& f) {
  if (dtype == DT_VOL_F32) f(float{});
  else if (dtype == DT_VOL_F16) f(__half{});
  else f(__hip_bfloat16{});
}

// the mask as the kernels with the planes innermost read it
template <typename F>
void by_mask(const uint8_t* mask, int64_t plane_stride, F&& f) {
  if (!mask || plane_stride == 0) f(std::integral_constant<MaskKind, kNoMask>{});
  else if (plane_stride == 1) f(std::integral_constant<MaskKind, kMaskVectors>{});
  else f(std::integral_constant<MaskKind, kMaskBytes>{});
}

// lists of 0, 1, 4 and 8 slots
template <typename F>
void by_top(int top, F&& f) {
  if (top == 0) f(std::integral_constant<int, 0>{});
  else if (top == 1) f(std::integral_constant<int, 1>{});
  else if (top <= 4) f(std::integral_constant<int, 4>{});
  else f(std::integral_constant<int, 8>{});
}

// bytes from a tensor's first pixel to its last (and over `planes` planes)
int64_t span_of(const int64_t (&s)[4], int b, int h, int w, int64_t planes, int size) {
  return ((b - 1) * s[0] + (h - 1) * s[2] + (w - 1) * s[3] + planes * s[1]) * size;
}
constexpr int64_t kNear = (int64_t)1 << 32;

// Four lanes per pixel, in launches of at most 2^29 pixels: from 2^30 on a single one would have 2^32 work items, more than a grid takes.
// (With 32-bit offsets a volume has fewer than 2^29 pixels, kNear / 8.)
template <typename A, typename F>
void by_range(A a, F&& launch) {
  constexpr uint32_t kRange = 1u << 29;
  const uint32_t pixels = (uint32_t)a.b * a.h * a.w;
  for (a.first = 0; a.first < pixels; a.first += kRange) launch(a, dim3((std::min(pixels - a.first, kRange) + 63) / 64));
}

template <typename T, int K>
void launch_stats(const PlaneFwd& a, hipStream_t s) {
  const uint32_t pixels = (uint32_t)a.b * a.h * a.w;
  const dim3 block(256), by_pixel((pixels + 255) / 256), by_four((pixels + 63) / 64);
  // Four waves per 64 pixels pay (the exchange, four lanes writing a pixel) where few pixels with many planes would leave the chip idle.
  // Measured us, fp32, 0 / 4 alternatives, four waves against one:
  //   D = 16:   19200 pixels  4.2 /  4.9 against  3.2 /  4.2; 307200 pixels 13.8 / 19.8 against  6.3 / 10.0
  //   D = 64:   76800 pixels  6.7 /  9.1 against  7.1 / 10.8; 307200 pixels 17.0 / 24.3 against 17.0 / 21.1
  //   D = 128: 153600 pixels 15.4 / 21.2 against 15.7 / 24.2; 307200 pixels 32.0 / 41.1 against 31.8 / 39.7
  const bool share = (int64_t)pixels < 2400 * ((int64_t)a.d - 24);
  if (a.vs[1] == 1)
    by_mask(a.mask, a.ms[1], [&](auto m) { DT_LAUNCH((plane_stats_last_kernel<T, K, m.value, uint32_t>), by_four, block, 0, s, a); });
  else if (share) DT_LAUNCH((plane_stats_first_kernel<T, K, 4, uint32_t>), by_four, block, 0, s, a);
  else DT_LAUNCH((plane_stats_first_kernel<T, K, 1, uint32_t>), by_pixel, block, 0, s, a);
}

// Volumes, masks or outputs beyond 32-bit offsets: one kernel per layout and kind of mask, with 8 slots whatever top is.  Per byte that costs
// little with alternatives and more without: float16, 57 x 128 x 480 x 640 (4.5 GB) against 48 of them (3.8 GB) with 32-bit offsets, us
// per batch element: pixels innermost 29.1 against 25.4 with 4, 27.7 against 17.4 without; planes innermost 33.8 / 27.6 and 31.9 / 17.9.
template <typename T>
void launch_stats_wide(const PlaneFwd& a, hipStream_t s) {
  const uint32_t pixels = (uint32_t)a.b * a.h * a.w;
  if (a.vs[1] == 1)
    by_mask(a.mask, a.ms[1], [&](auto m) {
      by_range(a, [&](const PlaneFwd& r, dim3 grid) { DT_LAUNCH((plane_stats_last_kernel<T, 8, m.value, int64_t>), grid, dim3(256), 0, s, r); });
    });
  else DT_LAUNCH((plane_stats_first_kernel<T, 8, 1, int64_t>), dim3((pixels + 255) / 256), dim3(256), 0, s, a);
}

template <typename T, int K, typename Off>
void launch_grad(const PlaneBwd& a, hipStream_t s) {
  const uint32_t pixels = (uint32_t)a.b * a.h * a.w;
  const dim3 block(256), by_pixel((pixels + 255) / 256, std::min(65535, (a.d + kN - 1) / kN));
  if (a.vs[1] == 1 && a.gs[1] == 1) {
    by_range(a, [&](const PlaneBwd& r, dim3 grid) {
      // (bytes also where they lie next to each other: the vectors cost this kernel twice the registers)
      if (a.mask && a.ms[1] != 0) DT_LAUNCH((plane_grad_last_kernel<T, K, kMaskBytes, Off>), grid, block, 0, s, r);
      else DT_LAUNCH((plane_grad_last_kernel<T, K, kNoMask, Off>), grid, block, 0, s, r);
    });
  } else {
    DT_LAUNCH((plane_grad_first_kernel<T, K, Off>), by_pixel, block, 0, s, a);
  }
}

int check_desc(const char* what, const dt_plane_desc* d) {
  DT_REQUIRE(d, "%s: null descriptor", what);
  DT_REQUIRE(d->b > 0 && d->d > 0 && d->d <= DT_PLANE_MAX_PLANES && d->h > 0 && d->w > 0, "%s: bad extents b=%d d=%d h=%d w=%d", what, d->b, d->d, d->h, d->w);
  DT_REQUIRE((int64_t)d->b * d->h < INT32_MAX && (int64_t)d->b * d->h * d->w < INT32_MAX, "%s: more than 2^31 - 1 pixels", what);
  DT_REQUIRE(d->dtype == DT_VOL_F32 || d->dtype == DT_VOL_F16 || d->dtype == DT_VOL_BF16, "%s: unknown dtype %d", what, d->dtype);
  DT_REQUIRE(d->top >= 0 && d->top <= DT_PLANE_MAX_TOP && d->top <= d->d, "%s: top=%d not in 0..%d", what, d->top,
             d->d < DT_PLANE_MAX_TOP ? d->d : DT_PLANE_MAX_TOP);
  // (scale log2 e and the gradient's scale * g * log probability have to be finite)
  DT_REQUIRE(d->scale >= 0.999e-30f && d->scale <= 1.001e30f, "%s: scale=%g not in 1e-30..1e30", what, (double)d->scale);
  for (int i = 0; i < 4; ++i)
    DT_REQUIRE(d->vol_stride[i] >= 0 && d->mask_stride[i] >= 0 && d->planes_stride[i] >= 0 && d->grad_stride[i] >= 0,
               "%s: negative stride", what);
  return 0;
}

}  // namespace dt

using namespace dt;

extern "C" {

int dt_cv_plane_log_probs(const dt_plane_desc* d, const void* volume, const uint8_t* mask, const int64_t* plane_bhw,
                          const float* depth_planes, float* log_prob, float* entropy, float* log_sum, float* top_log_prob,
                          int64_t* top_plane, float* top_depth, float* row_max, float* row_log, dt_stream_t s) {
  if (check_desc("dt_cv_plane_log_probs", d)) return 1;
  DT_REQUIRE(volume && entropy && log_sum, "dt_cv_plane_log_probs: null pointer");
  DT_REQUIRE(!plane_bhw == !log_prob, "dt_cv_plane_log_probs: log_prob goes with plane_bhw");
  DT_REQUIRE(d->top == 0 || (top_log_prob && top_plane), "dt_cv_plane_log_probs: top=%d without its outputs", d->top);
  DT_REQUIRE(!top_depth || (depth_planes && d->top), "dt_cv_plane_log_probs: top_depth without depth_planes or alternatives");
  DT_REQUIRE(!row_max == !row_log, "dt_cv_plane_log_probs: row_max goes with row_log");
  PlaneFwd a{volume, mask, plane_bhw, depth_planes, log_prob, entropy, log_sum, top_log_prob, top_plane, top_depth, row_max, row_log};
  for (int i = 0; i < 4; ++i) a.vs[i] = d->vol_stride[i], a.ms[i] = d->mask_stride[i], a.ps[i] = d->planes_stride[i];
  a.b = d->b, a.d = d->d, a.h = d->h, a.w = d->w, a.top = d->top, a.scale = d->scale, a.outside = d->outside;
  a.by_hw = make_div((uint32_t)d->h * d->w), a.by_w = make_div(d->w);
  by_type(d->dtype, [&](auto v) {
    const bool last = a.vs[1] == 1;
    if (span_of(a.vs, a.b, a.h, a.w, last ? a.d : 0, sizeof v) >= kNear || (mask && span_of(a.ms, a.b, a.h, a.w, last ? a.d : 0, 1) >= kNear) ||
        (a.top_depth && span_of(a.ps, a.b, a.h, a.w, a.d, 4) >= kNear) || (int64_t)a.b * std::max(a.top, 1) * a.h * a.w >= kNear / 8)
      launch_stats_wide<decltype(v)>(a, to_stream(s));
    else
      by_top(a.top, [&](auto k) { launch_stats<decltype(v), k.value>(a, to_stream(s)); });
  });
  return check_launch("dt_cv_plane_log_probs");
}

int dt_cv_plane_log_probs_grad(const dt_plane_desc* d, const void* volume, const uint8_t* mask, const int64_t* plane_bhw,
                               const float* entropy, const int64_t* top_plane, const float* row_max, const float* row_log,
                               const float* g_log_prob, const float* g_entropy, const float* g_log_sum, const float* g_top_log_prob,
                               void* grad_volume, dt_stream_t s) {
  if (check_desc("dt_cv_plane_log_probs_grad", d)) return 1;
  DT_REQUIRE(volume && entropy && row_max && row_log && grad_volume, "dt_cv_plane_log_probs_grad: null pointer");
  DT_REQUIRE(!g_log_prob || plane_bhw, "dt_cv_plane_log_probs_grad: g_log_prob without plane_bhw");
  DT_REQUIRE(!g_top_log_prob || (d->top && top_plane), "dt_cv_plane_log_probs_grad: g_top_log_prob without top_plane");
  PlaneBwd a{volume, mask, plane_bhw, entropy, top_plane, row_max, row_log, g_log_prob, g_entropy, g_log_sum, g_top_log_prob, grad_volume};
  for (int i = 0; i < 4; ++i) a.vs[i] = d->vol_stride[i], a.ms[i] = d->mask_stride[i], a.gs[i] = d->grad_stride[i];
  a.b = d->b, a.d = d->d, a.h = d->h, a.w = d->w, a.top = d->top, a.scale = d->scale;
  a.by_hw = make_div((uint32_t)d->h * d->w), a.by_w = make_div(d->w);
  if (!g_top_log_prob) a.top = 0;
  by_type(d->dtype, [&](auto v) {
    const bool last = a.vs[1] == 1 && a.gs[1] == 1;
    const bool wide = span_of(a.vs, a.b, a.h, a.w, last ? a.d : 0, sizeof v) >= kNear ||
                      span_of(a.gs, a.b, a.h, a.w, last ? a.d : 0, sizeof v) >= kNear ||
                      (mask && span_of(a.ms, a.b, a.h, a.w, last ? a.d : 0, 1) >= kNear) ||
                      (int64_t)a.b * std::max(a.top, 1) * a.h * a.w >= kNear / 8;
    if (wide) launch_grad<decltype(v), 8, int64_t>(a, to_stream(s));
    else by_top(a.top, [&](auto k) { launch_grad<decltype(v), k.value, uint32_t>(a, to_stream(s)); });
  });
  return check_launch("dt_cv_plane_log_probs_grad");
}

int dt_cv_nearest_planes_f32(const float* depth_bhw, const float* depth_planes, const int64_t* planes_stride4, int b, int d, int h,
                             int w, int64_t* plane_bhw, dt_stream_t s) {
  DT_REQUIRE(b > 0 && d > 0 && d <= DT_PLANE_MAX_NEAREST && h > 0 && w > 0, "dt_cv_nearest_planes_f32: bad extents b=%d d=%d h=%d w=%d", b, d, h, w);
  DT_REQUIRE((int64_t)b * h < INT32_MAX && (int64_t)b * h * w < INT32_MAX, "dt_cv_nearest_planes_f32: more than 2^31 - 1 pixels");
  DT_REQUIRE(depth_bhw && depth_planes && planes_stride4 && plane_bhw, "dt_cv_nearest_planes_f32: null pointer");
  PlaneNear a{depth_bhw, depth_planes, plane_bhw};
  for (int i = 0; i < 4; ++i) {
    DT_REQUIRE(planes_stride4[i] >= 0, "dt_cv_nearest_planes_f32: negative stride");
    a.ps[i] = planes_stride4[i];
  }
  a.b = b, a.d = d, a.h = h, a.w = w;
  a.by_hw = make_div((uint32_t)h * w), a.by_w = make_div(w);
  const unsigned pixels = (unsigned)b * h * w;
  DT_LAUNCH(nearest_planes_kernel, dim3((pixels + 63) / 64), dim3(64), 0, to_stream(s), a);
  return check_launch("dt_cv_nearest_planes_f32");
}

}  // extern "C"
