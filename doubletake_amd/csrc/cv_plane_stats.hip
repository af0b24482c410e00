// The plane-sweep volume read as a distribution over depth planes: log probability of a given plane, entropy, normaliser and the
// most probable planes of every pixel; the gradient of the volume for gradients of these; the plane index of a metric depth.
// Formulas and edge cases: include/doubletake_hip.h.
#include "common.hpp"

#include <hip/hip_fp16.h>
#include <hip/hip_bf16.h>
#include <cmath>

namespace dt {

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
  float scale;
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
  int b, y, x;
};
__device__ __forceinline__ Pixel pixel_of(unsigned p, int h, int w) {
  const unsigned row = p / (unsigned)w;
  Pixel q;
  q.x = (int)(p - row * (unsigned)w);
  q.b = (int)(row / (unsigned)h);
  q.y = (int)(row - (unsigned)q.b * (unsigned)h);
  return q;
}
__device__ __forceinline__ int64_t offset_of(const int64_t (&s)[4], const Pixel& q) { return q.b * s[0] + q.y * s[2] + q.x * s[3]; }

// scale (x - m) - ls for the outputs: halves, so that two scores at opposite ends of the float range do not overflow in between
__device__ __forceinline__ float log_prob_of(float x, float m, float ls, float scale) {
  return 2.f * ((0.5f * x - 0.5f * m) * scale) - ls;
}

// a before b among the alternatives: the larger score, NaN above everything, the lower plane of equals
__device__ __forceinline__ bool ranks_above(float a, int ia, float b, int ib) {
  const bool na = a != a, nb = b != b;
  if (na != nb) return na;
  if (!na && a != b) return a > b;
  return (unsigned)ia < (unsigned)ib;  // (-1, an empty slot, ranks last)
}

template <typename T>
__global__ void __launch_bounds__(256) plane_stats_kernel(PlaneFwd a) {
  const unsigned p = blockIdx.x * 256u + threadIdx.x;
  if (p >= (unsigned)a.b * a.h * a.w) return;
  const Pixel q = pixel_of(p, a.h, a.w);
  const T* vol = (const T*)a.vol + offset_of(a.vs, q);
  const uint8_t* mask = a.mask ? a.mask + offset_of(a.ms, q) : nullptr;
  auto score = [&](int d) { return mask && !mask[d * a.ms[1]] ? -INFINITY : to_f32(vol[d * a.vs[1]]); };
  float m = -INFINITY;
  float tv[DT_PLANE_MAX_TOP];
  int ti[DT_PLANE_MAX_TOP];
#pragma unroll
  for (int j = 0; j < DT_PLANE_MAX_TOP; ++j) tv[j] = -INFINITY, ti[j] = -1;
  for (int d = 0; d < a.d; ++d) {
    float x = score(d);
    m = fmaxf(m, x);
    if (x == -INFINITY) continue;
    int i = d;
#pragma unroll
    for (int j = 0; j < DT_PLANE_MAX_TOP; ++j) {
      const bool take = ti[j] < 0 || ranks_above(x, i, tv[j], ti[j]);
      const float xv = tv[j];
      const int xi = ti[j];
      tv[j] = take ? x : xv, ti[j] = take ? i : xi;
      x = take ? xv : x, i = take ? xi : i;
    }
  }
  const float m0 = m == -INFINITY ? 0.f : m;
  float s = 0.f, t = 0.f;
  for (int d = 0; d < a.d; ++d) {
    const float y = a.scale * (score(d) - m0);
    const float e = expf(y);
    s += e;
    t += e * fmaxf(y, -1e4f);
  }
  const bool empty = s == 0.f;
  const float ls = logf(s);
  a.entropy[p] = empty ? 0.f : ls - t / s;
  a.log_sum[p] = m0 * a.scale + ls;
  if (a.row_max) a.row_max[p] = m0, a.row_log[p] = ls;
  if (a.plane) {
    const int64_t g = a.plane[p];
    a.log_prob[p] = g < 0 || g >= a.d ? 0.f : empty ? -INFINITY : log_prob_of(score((int)g), m0, ls, a.scale);
  }
  const size_t hw = (size_t)a.h * a.w;
  const size_t o = (size_t)q.b * a.top * hw + (size_t)q.y * a.w + q.x;
#pragma unroll
  for (int j = 0; j < DT_PLANE_MAX_TOP; ++j) {
    if (j >= a.top) break;
    a.top_plane[o + j * hw] = ti[j];
    a.top_log_prob[o + j * hw] = ti[j] < 0 ? -INFINITY : log_prob_of(tv[j], m0, ls, a.scale);
    if (a.top_depth) a.top_depth[o + j * hw] = ti[j] < 0 ? 0.f : a.planes[offset_of(a.ps, q) + ti[j] * a.ps[1]];
  }
}

template <typename T>
__global__ void __launch_bounds__(256) plane_grad_kernel(PlaneBwd a) {
  const unsigned p = blockIdx.x * 256u + threadIdx.x;
  if (p >= (unsigned)a.b * a.h * a.w) return;
  const Pixel q = pixel_of(p, a.h, a.w);
  const T* vol = (const T*)a.vol + offset_of(a.vs, q);
  T* grad = (T*)a.grad + offset_of(a.gs, q);
  const uint8_t* mask = a.mask ? a.mask + offset_of(a.ms, q) : nullptr;
  const float m = a.row_max[p], ls = a.row_log[p], ent = a.entropy[p];
  const bool empty = ls == -INFINITY;
  const float ge = a.g_entropy ? a.g_entropy[p] : 0.f;
  float all = a.g_log_sum ? a.g_log_sum[p] : 0.f;
  int hit = -1;
  float gl = 0.f;
  if (a.g_log_prob) {
    const int64_t g = a.plane[p];
    if (g >= 0 && g < a.d) hit = (int)g, gl = a.g_log_prob[p], all -= gl;
  }
  int ti[DT_PLANE_MAX_TOP];
  float tg[DT_PLANE_MAX_TOP];
  const size_t hw = (size_t)a.h * a.w;
  const size_t o = (size_t)q.b * a.top * hw + (size_t)q.y * a.w + q.x;
#pragma unroll
  for (int j = 0; j < DT_PLANE_MAX_TOP; ++j) {
    ti[j] = -1, tg[j] = 0.f;
    if (a.g_top && j < a.top) {
      ti[j] = (int)a.top_plane[o + j * hw];
      if (ti[j] >= 0) tg[j] = a.g_top[o + j * hw], all -= tg[j];
    }
  }
  for (int d = 0; d < a.d; ++d) {
    const float x = to_f32(vol[d * a.vs[1]]);
    float g = 0.f;
    if (!empty && !(mask && !mask[d * a.ms[1]]) && x != -INFINITY) {
      const float lp = a.scale * (x - m) - ls;
      const float pr = expf(lp);
      g = pr * (all - ge * (fmaxf(lp, -1e4f) + ent));
      if (d == hit) g += gl;
#pragma unroll
      for (int j = 0; j < DT_PLANE_MAX_TOP; ++j)
        if (d == ti[j]) g += tg[j];
    }
    grad[d * a.gs[1]] = from_f32<T>(a.scale * g);
  }
}

__global__ void __launch_bounds__(256) nearest_planes_kernel(PlaneNear a) {
  const unsigned p = blockIdx.x * 256u + threadIdx.x;
  if (p >= (unsigned)a.b * a.h * a.w) return;
  const Pixel q = pixel_of(p, a.h, a.w);
  const float* planes = a.planes + offset_of(a.ps, q);
  const float depth = a.depth[p];
  int at = -1;
  if (depth > 0.f && depth < INFINITY) {
    double best = INFINITY;
    for (int d = 0; d < a.d; ++d) {
      const double off = fabs((double)planes[d * a.ps[1]] - (double)depth);
      if (off < best) best = off, at = d;
    }
  }
  a.out[p] = at;
}

template <typename F>
int by_type(int dtype, F&& f) {
  switch (dtype) {
    case DT_VOL_F32: return f(float{});
    case DT_VOL_F16: return f(__half{});
    default: return f(__hip_bfloat16{});
  }
}

int check_desc(const char* what, const dt_plane_desc* d) {
  DT_REQUIRE(d, "%s: null descriptor", what);
  DT_REQUIRE(d->b > 0 && d->d > 0 && d->h > 0 && d->w > 0, "%s: bad extents b=%d d=%d h=%d w=%d", what, d->b, d->d, d->h, d->w);
  DT_REQUIRE((int64_t)d->b * d->h < INT32_MAX && (int64_t)d->b * d->h * d->w < INT32_MAX, "%s: more than 2^31 - 1 pixels", what);
  DT_REQUIRE(d->dtype == DT_VOL_F32 || d->dtype == DT_VOL_F16 || d->dtype == DT_VOL_BF16, "%s: unknown dtype %d", what, d->dtype);
  DT_REQUIRE(d->top >= 0 && d->top <= DT_PLANE_MAX_TOP && d->top <= d->d, "%s: top=%d not in 0..%d", what, d->top,
             d->d < DT_PLANE_MAX_TOP ? d->d : DT_PLANE_MAX_TOP);
  DT_REQUIRE(d->scale > 0.f && std::isfinite(d->scale), "%s: scale=%g is not positive and finite", what, (double)d->scale);
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
  a.b = d->b, a.d = d->d, a.h = d->h, a.w = d->w, a.top = d->top, a.scale = d->scale;
  const unsigned pixels = (unsigned)d->b * d->h * d->w;
  return by_type(d->dtype, [&](auto v) {
    DT_LAUNCH(plane_stats_kernel<decltype(v)>, dim3((pixels + 255) / 256), dim3(256), 0, to_stream(s), a);
    return check_launch("dt_cv_plane_log_probs");
  });
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
  const unsigned pixels = (unsigned)d->b * d->h * d->w;
  return by_type(d->dtype, [&](auto v) {
    DT_LAUNCH(plane_grad_kernel<decltype(v)>, dim3((pixels + 255) / 256), dim3(256), 0, to_stream(s), a);
    return check_launch("dt_cv_plane_log_probs_grad");
  });
}

int dt_cv_nearest_planes_f32(const float* depth_bhw, const float* depth_planes, const int64_t* planes_stride4, int b, int d, int h,
                             int w, int64_t* plane_bhw, dt_stream_t s) {
  DT_REQUIRE(b > 0 && d > 0 && h > 0 && w > 0, "dt_cv_nearest_planes_f32: bad extents b=%d d=%d h=%d w=%d", b, d, h, w);
  DT_REQUIRE((int64_t)b * h < INT32_MAX && (int64_t)b * h * w < INT32_MAX, "dt_cv_nearest_planes_f32: more than 2^31 - 1 pixels");
  DT_REQUIRE(depth_bhw && depth_planes && planes_stride4 && plane_bhw, "dt_cv_nearest_planes_f32: null pointer");
  PlaneNear a{depth_bhw, depth_planes, plane_bhw};
  for (int i = 0; i < 4; ++i) a.ps[i] = planes_stride4[i];
  a.b = b, a.d = d, a.h = h, a.w = w;
  const unsigned pixels = (unsigned)b * h * w;
  DT_LAUNCH(nearest_planes_kernel, dim3((pixels + 255) / 256), dim3(256), 0, to_stream(s), a);
  return check_launch("dt_cv_nearest_planes_f32");
}

}  // extern "C"
