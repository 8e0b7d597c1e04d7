// lqg_adamw.hip — one AdamW step over many tensors, moments in float / double or in 8 bits (include/lqg_learn.h).
//
// Memory bound: an element of a float tensor moves 28 bytes (p, m, v read and written, g read), 16 with 8-bit moments.  One launch
// walks up to TENSORS tensors: their table travels in the kernel's arguments, so that no table has to be copied to the device and kept
// alive; a workgroup finds its tensor by bisection in uniform (scalar) registers.  This file is compiled with -ffp-contract=off: every
// operation rounds by itself, so a step gives the bits that the same formula gives written operation by operation.
#include "lqg_learn.hpp"

#include <cmath>

using namespace lqg::learn;

namespace {

constexpr int TENSORS = 96;      // 3.5 kB of arguments
constexpr int CHUNK = 2048;      // elements of a workgroup: 256 lanes x 2 vectors of 4
constexpr int BLOCK = 256;       // elements that share a scale (8 bits): a wave, 4 per lane
constexpr float F8_MAX = 448.0f, TINY = 1e-30f, LEAST = 0x1p-9f;

struct Table {
  int32_t count;
  int32_t start[TENSORS + 1];    // first chunk of each tensor
  void* p[TENSORS];
  const void* g[TENSORS];
  int64_t n[TENSORS], off[TENSORS];
};

template <class S> struct Hyper {
  S b1, a1, b2, a2, decay, lr, eps, inv1, inv2;     // a1 = 1 - b1, inv1 = 1 / (1 - b1^t)
  const double* state;                              // {t, inv1, inv2} or NULL
};

template <class T> struct alignas(4 * sizeof(T)) Vec4 { T v[4]; };

template <class S> __device__ inline S root(S x);
template <> __device__ inline float root(float x) { return sqrtf(x); }
template <> __device__ inline double root(double x) { return sqrt(x); }

template <class S> __device__ inline void moments(const Hyper<S>& h, S g, S& m, S& v) {
  m = h.b1 * m + h.a1 * g;
  v = h.b2 * v + (h.a2 * g) * g;
}
template <class S> __device__ inline S moved(const Hyper<S>& h, S inv1, S inv2, S p, S m, S v) {
  const S far = root<S>(v * inv2) + h.eps;
  return p * h.decay - (h.lr * (m * inv1)) / far;
}

__device__ inline int tensor_of(const Table& t, int chunk) {
  int lo = 0, hi = t.count - 1;                     // the last tensor that starts at or before the chunk
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (t.start[mid] <= chunk) lo = mid;
    else hi = mid - 1;
  }
  return lo;
}

// four elements at i, of which `left` exist; whole: the pointer is aligned for a vector
template <class T> __device__ inline Vec4<T> load4(const T* p, bool whole, long left) {
  if (whole && left >= 4) return *reinterpret_cast<const Vec4<T>*>(p);
  Vec4<T> r;
#pragma unroll
  for (int k = 0; k < 4; ++k) r.v[k] = k < left ? p[k] : (T)0.0f;
  return r;
}
template <class T> __device__ inline void store4(T* p, const Vec4<T>& r, bool whole, long left) {
  if (whole && left >= 4) {
    *reinterpret_cast<Vec4<T>*>(p) = r;
    return;
  }
#pragma unroll
  for (int k = 0; k < 4; ++k)
    if (k < left) p[k] = r.v[k];
}

// T: tensors' type, S: type of the moments and of the arithmetic
template <class T, class S>
__global__ __launch_bounds__(256) void k_adamw(const Table tab, const Hyper<S> h, S* ms, S* vs) {
  const int i = tensor_of(tab, (int)blockIdx.x);
  const long at = (long)((int)blockIdx.x - tab.start[i]) * CHUNK + threadIdx.x * 4, n = tab.n[i];
  T* p = static_cast<T*>(tab.p[i]);
  const T* g = static_cast<const T*>(tab.g[i]);
  const bool whole = (((uintptr_t)p | (uintptr_t)g) & (sizeof(T) * 4 - 1)) == 0;
  S* m = ms + tab.off[i];
  S* v = vs + tab.off[i];
  const S inv1 = h.state ? (S)h.state[1] : h.inv1, inv2 = h.state ? (S)h.state[2] : h.inv2;
  Vec4<T> pv[2], gv[2];
  Vec4<S> mv[2], vv[2];
#pragma unroll
  for (int q = 0; q < 2; ++q) {
    const long e = at + q * 1024, left = n - e;
    if (left <= 0) continue;
    pv[q] = load4(p + e, whole, left);
    gv[q] = load4(g + e, whole, left);
    mv[q] = load4(m + e, true, left);
    vv[q] = load4(v + e, true, left);
  }
#pragma unroll
  for (int q = 0; q < 2; ++q) {
    const long e = at + q * 1024, left = n - e;
    if (left <= 0) continue;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      moments<S>(h, (S)gv[q].v[k], mv[q].v[k], vv[q].v[k]);
      pv[q].v[k] = (T)moved<S>(h, inv1, inv2, (S)pv[q].v[k], mv[q].v[k], vv[q].v[k]);
    }
    store4(p + e, pv[q], whole, left);
    store4(m + e, mv[q], true, left);
    store4(v + e, vv[q], true, left);
  }
}

// largest of the bit patterns of |x| over the wave: orders magnitudes, and puts a NaN above them all
__device__ inline uint32_t wave_top(uint32_t x) {
#pragma unroll
  for (int k = 1; k < 64; k <<= 1) x = max(x, (uint32_t)__shfl_xor((int)x, k));
  return x;
}
__device__ inline uint32_t top4(const float (&x)[4]) {
  uint32_t t = 0;
#pragma unroll
  for (int k = 0; k < 4; ++k) t = max(t, __float_as_uint(x[k]) & 0x7fffffffu);
  return wave_top(t);
}
__device__ inline void unpack(uint32_t c, float scale, float (&x)[4]) {
  const auto lo = __builtin_amdgcn_cvt_pk_f32_fp8((int)c, false), hi = __builtin_amdgcn_cvt_pk_f32_fp8((int)c, true);
  x[0] = lo[0] * scale, x[1] = lo[1] * scale, x[2] = hi[0] * scale, x[3] = hi[1] * scale;
}
__device__ inline uint32_t pack(const float (&x)[4]) {
  int c = __builtin_amdgcn_cvt_pk_fp8_f32(x[0], x[1], 0, false);
  return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(x[2], x[3], c, true);
}

template <class T>
__global__ __launch_bounds__(256) void k_adamw8(const Table tab, const Hyper<float> h, uint32_t* ms, uint32_t* rs, float* m_scale,
                                                float* r_scale) {
  const int i = tensor_of(tab, (int)blockIdx.x);
  const long n = tab.n[i];
  T* p = static_cast<T*>(tab.p[i]);
  const T* g = static_cast<const T*>(tab.g[i]);
  const bool whole = (((uintptr_t)p | (uintptr_t)g) & (sizeof(T) * 4 - 1)) == 0;
  const float inv1 = h.state ? (float)h.state[1] : h.inv1, inv2 = h.state ? (float)h.state[2] : h.inv2;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const long first = (long)((int)blockIdx.x - tab.start[i]) * CHUNK;
#pragma unroll
  for (int q = 0; q < 2; ++q) {
    const long e0 = first + (q * 4 + wave) * BLOCK;          // the wave's block; uniform in the wave
    if (e0 >= n) continue;
    const long e = e0 + lane * 4, left = n - e, o = tab.off[i] + e;
    const long sc = (tab.off[i] + e0) / BLOCK;
    float m[4], r[4], v[4], pf[4];
    unpack(ms[o / 4], m_scale[sc], m);
    unpack(rs[o / 4], r_scale[sc], r);
    Vec4<T> pv, gv;
#pragma unroll
    for (int k = 0; k < 4; ++k) pv.v[k] = (T)0.0f, gv.v[k] = (T)0.0f;
    if (left > 0) {
      pv = load4(p + e, whole, left);
      gv = load4(g + e, whole, left);
    }
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      v[k] = r[k] * r[k];
      moments<float>(h, (float)gv.v[k], m[k], v[k]);
      pf[k] = moved<float>(h, inv1, inv2, (float)pv.v[k], m[k], v[k]);
      r[k] = sqrtf(v[k]);
      if (k >= left) m[k] = 0.0f, r[k] = 0.0f;               // behind the tensor's end
      pv.v[k] = (T)pf[k];
    }
    const float mt = __uint_as_float(top4(m)), rt = __uint_as_float(top4(r));
    const bool mz = mt < TINY, rz = rt < TINY;               // (false for a NaN, which then reaches the codes)
    const float mi = mz ? 0.0f : F8_MAX / mt, ri = rz ? 0.0f : F8_MAX / rt;
    float mc[4], rc[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      mc[k] = m[k] * mi;
      rc[k] = r[k] * ri;
      // (half the least value, ties to even: what is at most that rounds to 0)
      if (r[k] > 0.0f && rc[k] < LEAST && !rz) rc[k] = LEAST;
    }
    if (left > 0) store4(p + e, pv, whole, left);
    ms[o / 4] = pack(mc);
    rs[o / 4] = pack(rc);
    if (lane == 0) {
      m_scale[sc] = mz ? 0.0f : mt / F8_MAX;
      r_scale[sc] = rz ? 0.0f : rt / F8_MAX;
    }
  }
}

__global__ void k_advance(double* s, double b1, double b2) {
  const double t = s[0] + 1.0;
  s[0] = t;
  s[1] = 1.0 / (1.0 - pow(b1, t));
  s[2] = 1.0 / (1.0 - pow(b2, t));
}

template <class S> Hyper<S> hyper(const lqg_adamw* p) {
  Hyper<S> h;
  h.b1 = (S)p->beta1, h.a1 = (S)(1.0 - p->beta1), h.b2 = (S)p->beta2, h.a2 = (S)(1.0 - p->beta2);
  h.decay = (S)(1.0 - p->lr * p->weight_decay), h.lr = (S)p->lr, h.eps = (S)p->eps;
  const double t = (double)p->step;
  h.inv1 = (S)1 / (S)(1.0 - std::pow(p->beta1, t)), h.inv2 = (S)1 / (S)(1.0 - std::pow(p->beta2, t));
  h.state = p->step_state;
  return h;
}

template <class T, class S> void launch(const lqg_adamw* p, const Table& t, hipStream_t st) {
  const unsigned groups = (unsigned)t.start[t.count];
  if constexpr (sizeof(S) == 4) {
    if (p->bits == 8) {
      hipLaunchKernelGGL((k_adamw8<T>), dim3(groups), dim3(256), 0, st, t, hyper<float>(p), static_cast<uint32_t*>(p->exp_avg),
                         static_cast<uint32_t*>(p->exp_avg_sq), p->exp_avg_scale, p->exp_avg_sq_scale);
      return;
    }
  }
  hipLaunchKernelGGL((k_adamw<T, S>), dim3(groups), dim3(256), 0, st, t, hyper<S>(p), static_cast<S*>(p->exp_avg),
                     static_cast<S*>(p->exp_avg_sq));
}

}  // namespace

extern "C" int lqg_adamw_step(const lqg_adamw* p, void* stream) {
  if (!p || !p->params || !p->grads || !p->numel || !p->offset || !p->exp_avg || !p->exp_avg_sq) return LQG_ERR_NULL;
  if (p->count < 0 || (p->bits != 8 && p->bits != 32) || p->type < LQG_T_F32 || p->type > LQG_T_F64) return LQG_ERR_ARG;
  if (p->bits == 8 && (p->type == LQG_T_F64 || !p->exp_avg_scale || !p->exp_avg_sq_scale)) return LQG_ERR_ARG;
  if (!p->step_state && p->step < 1) return LQG_ERR_ARG;
  for (int i = 0; i < p->count; ++i) {
    if (p->numel[i] < 0 || p->offset[i] < 0 || p->offset[i] % BLOCK) return LQG_ERR_ARG;
    if (p->numel[i] && (!p->params[i] || !p->grads[i])) return LQG_ERR_NULL;
    const long chunks = (p->numel[i] + CHUNK - 1) / CHUNK;
    if (!grid_fits(chunks + 1, 256)) return LQG_ERR_ARG;
  }
  Table t;
  t.count = 0;
  t.start[0] = 0;
  auto flush = [&]() {
    if (!t.count) return 0;
    hipStream_t st = (hipStream_t)stream;
    if (p->type == LQG_T_F32) launch<float, float>(p, t, st);
    else if (p->type == LQG_T_BF16) launch<bf16, float>(p, t, st);
    else if (p->type == LQG_T_F16) launch<f16, float>(p, t, st);
    else launch<double, double>(p, t, st);
    t.count = 0;
    return (int)last();
  };
  for (int i = 0; i < p->count; ++i) {
    if (!p->numel[i]) continue;
    const long chunks = (p->numel[i] + CHUNK - 1) / CHUNK;
    if (t.count == TENSORS || (t.count && !grid_fits(t.start[t.count] + chunks, 256)))
      if (const int rc = flush()) return rc;
    t.p[t.count] = p->params[i];
    t.g[t.count] = p->grads[i];
    t.n[t.count] = p->numel[i];
    t.off[t.count] = p->offset[i];
    t.start[t.count + 1] = t.start[t.count] + (int32_t)chunks;
    ++t.count;
  }
  return flush();
}

extern "C" int lqg_adamw_advance(double* step_state, double beta1, double beta2, void* stream) {
  if (!step_state) return LQG_ERR_NULL;
  hipLaunchKernelGGL(k_advance, dim3(1), dim3(1), 0, (hipStream_t)stream, step_state, beta1, beta2);
  return (int)last();
}
