// lqg_conv.hip — short causal convolution over each channel, its gradients and its single step (include/lqg_learn.h).
//
// y[t] = act(bias + sum_k w[k] xs[t - (W-1) + k]).  Memory bound: 2 W (+ 6 for silu) flops per element read and written.  One lane walks
// one channel over a piece of the time axis with the last W rows in registers, so x is read once but for the W-1 rows before a piece.
#include "lqg_learn.hpp"

using namespace lqg::learn;

namespace {

constexpr int WMAX = 8;
constexpr int PIECE = 32;        // steps one lane walks (forward): (PIECE + W - 1) / PIECE rows read per row written
constexpr int GPIECE = 128;      // backward: longer, since each piece leaves W + 1 partial sums per channel

struct ConvArgs {
  lqg_conv p;
  long pieces, blocks;           // pieces of the time axis, blocks of 256 channels
  lqg_seq dy;
  const void *dstate_out;
  void *dx, *dstate;
  float* part;                   // [B * pieces][(W + 1)][D]
};

template <class T> __device__ inline const T* row(const lqg_seq& s, long b, long t) {
  return static_cast<const T*>(s.ptr) + b * s.sb + t * s.st;
}

__device__ inline long length_of(const int32_t* lengths, long b, long T) {
  if (!lengths) return T;
  const long n = lengths[b];
  return n < 0 ? 0 : (n > T ? T : n);
}

// row s of (state ++ x[:n]) counted from x's first step: state for s < 0
template <class T> __device__ inline float line(const ConvArgs& a, long b, long s, long d) {
  if (s >= 0) return up(row<T>(a.p.x, b, s)[d]);
  if (!a.p.state) return 0.0f;
  return up(static_cast<const T*>(a.p.state)[(b * (a.p.W - 1) + (s + a.p.W - 1)) * a.p.D + d]);
}

template <class T, int W>
__global__ __launch_bounds__(256) void k_conv(const ConvArgs a) {
  const long blk = blockIdx.x % a.blocks, rest = blockIdx.x / a.blocks;
  const long piece = rest % a.pieces, b = rest / a.pieces;
  const long d = blk * 256 + threadIdx.x;
  if (d >= a.p.D) return;
  const long n = length_of(a.p.lengths, b, a.p.T);
  const long t0 = piece * PIECE, t1 = min(t0 + PIECE, a.p.T);
  float w[W], r[W];
#pragma unroll
  for (int k = 0; k < W; ++k) w[k] = load_param(a.p.w, d * W + k);
  const float bias = a.p.bias.ptr ? load_param(a.p.bias, d) : 0.0f;
#pragma unroll
  for (int k = 1; k < W; ++k) r[k] = t0 < n ? line<T>(a, b, t0 - W + k, d) : 0.0f;     // rows t0-(W-1) .. t0-1
  T* y = static_cast<T*>(const_cast<void*>(a.p.y.ptr)) + b * a.p.y.sb + d;
#pragma unroll 4
  for (long t = t0; t < t1; ++t) {
#pragma unroll
    for (int k = 0; k + 1 < W; ++k) r[k] = r[k + 1];
    const bool live = t < n;
    r[W - 1] = live ? up(row<T>(a.p.x, b, t)[d]) : 0.0f;
    float v = bias;
#pragma unroll
    for (int k = 0; k < W; ++k) v = fmaf(w[k], r[k], v);
    if (a.p.silu) v *= sigmoid(v);
    y[t * a.p.y.st] = down<T>(live ? v : 0.0f);
  }
  if (a.p.state_out && piece == 0) {
    T* so = static_cast<T*>(a.p.state_out) + b * (W - 1) * a.p.D + d;
    for (int k = 0; k + 1 < W; ++k) so[k * a.p.D] = down<T>(line<T>(a, b, n - (W - 1) + k, d));
  }
}

// e[t] = dy[t] act'(v[t]);  dx[s] = sum_k w[k] e[s + W-1-k];  dw[k] = sum_t e[t] xs[t - (W-1) + k];  dbias = sum_t e[t].
// A lane recomputes v over its piece and the W-1 steps after it (whose e its last rows need), and finishes dx[t - (W-1)] at step t.
template <class T, int W>
__global__ __launch_bounds__(256) void k_conv_grad(const ConvArgs a) {
  const long blk = blockIdx.x % a.blocks, rest = blockIdx.x / a.blocks;
  const long piece = rest % a.pieces, b = rest / a.pieces;
  const long d = blk * 256 + threadIdx.x, D = a.p.D;
  if (d >= D) return;
  const long n = length_of(a.p.lengths, b, a.p.T);
  const long t0 = piece * GPIECE, t1 = min(t0 + GPIECE, a.p.T);
  float w[W], r[W], e[W], dw[W], db = 0.0f;
#pragma unroll
  for (int k = 0; k < W; ++k) w[k] = load_param(a.p.w, d * W + k), e[k] = 0.0f, dw[k] = 0.0f;
  const float bias = a.p.bias.ptr ? load_param(a.p.bias, d) : 0.0f;
#pragma unroll
  for (int k = 1; k < W; ++k) r[k] = t0 < n ? line<T>(a, b, t0 - W + k, d) : 0.0f;
  T* dx = static_cast<T*>(a.dx) + (b * a.p.T) * D + d;
  const T* so = static_cast<const T*>(a.dstate_out);
  // rows before the piece belong to the piece before it; the first piece owns the state's rows
  const long s0 = piece == 0 ? -(long)(W - 1) : t0;
  for (long t = t0; t < t1 + W - 1; ++t) {
#pragma unroll
    for (int k = 0; k + 1 < W; ++k) r[k] = r[k + 1], e[k] = e[k + 1];
    const bool live = t < n;
    r[W - 1] = live ? up(row<T>(a.p.x, b, t)[d]) : 0.0f;
    float g = live ? up(row<T>(a.dy, b, t)[d]) : 0.0f;
    if (a.p.silu) {
      float v = bias;
#pragma unroll
      for (int k = 0; k < W; ++k) v = fmaf(w[k], r[k], v);
      const float sg = sigmoid(v);
      g = live ? g * (sg * fmaf(v, 1.0f - sg, 1.0f)) : 0.0f;
    }
    e[W - 1] = g;
    if (t < t1 && live) {
      db += g;
#pragma unroll
      for (int k = 0; k < W; ++k) dw[k] = fmaf(g, r[k], dw[k]);
    }
    const long s = t - (W - 1);                  // e[0] = e[s] .. e[W-1] = e[s + W-1]
    if (s < s0) continue;
    float v = 0.0f;
#pragma unroll
    for (int k = 0; k < W; ++k) v = fmaf(w[k], e[W - 1 - k], v);
    if (so && s < n && s >= n - (W - 1)) v += up(so[(b * (W - 1) + (s - (n - (W - 1)))) * D + d]);
    if (s < 0) {
      if (a.dstate) static_cast<T*>(a.dstate)[(b * (W - 1) + s + W - 1) * D + d] = down<T>(v);
    } else {
      dx[s * D] = down<T>(s < n ? v : 0.0f);
    }
  }
  float* part = a.part + ((b * a.pieces + piece) * (W + 1)) * D + d;
#pragma unroll
  for (int k = 0; k < W; ++k) part[k * D] = dw[k];
  part[W * D] = db;
}

template <class T, int W>
__global__ __launch_bounds__(256) void k_conv_step(const ConvArgs a) {
  const long blk = blockIdx.x % a.blocks, b = blockIdx.x / a.blocks;
  const long d = blk * 256 + threadIdx.x, D = a.p.D;
  if (d >= D) return;
  T* st = static_cast<T*>(const_cast<void*>(a.p.state)) + b * (W - 1) * D + d;
  const T* x = static_cast<const T*>(a.p.x.ptr) + b * a.p.x.sb;
  T r[W];
#pragma unroll
  for (int k = 0; k + 1 < W; ++k) r[k] = st[k * D];
  r[W - 1] = x[d];
  float v = a.p.bias.ptr ? load_param(a.p.bias, d) : 0.0f;
#pragma unroll
  for (int k = 0; k < W; ++k) v = fmaf(load_param(a.p.w, d * W + k), up(r[k]), v);
  if (a.p.silu) v *= sigmoid(v);
  static_cast<T*>(const_cast<void*>(a.p.y.ptr))[b * a.p.y.sb + d] = down<T>(v);
#pragma unroll
  for (int k = 0; k + 1 < W; ++k) st[k * D] = r[k + 1];
}

// ------------------------------------------------------------------------------------------------ sums over rows
// 64 columns x 16 row lanes per workgroup: coalesced, and 16 independent chains of additions per column.
__global__ __launch_bounds__(1024) void k_row_sum_mid(const float* in, long rows, long cols, long outs, float* out) {
  __shared__ double s[16][64];
  const long blocks = (cols + 63) / 64;
  const long blk = blockIdx.x % blocks, o = blockIdx.x / blocks, c = blk * 64 + threadIdx.x;
  double v = 0.0;
  if (c < cols)
    for (long r = o + outs * threadIdx.y; r < rows; r += outs * 16) v += in[r * cols + c];
  s[threadIdx.y][threadIdx.x] = v;
  __syncthreads();
  if (threadIdx.y || c >= cols) return;
  v = 0.0;
#pragma unroll
  for (int k = 0; k < 16; ++k) v += s[k][threadIdx.x];
  out[o * cols + c] = (float)v;
}

__global__ __launch_bounds__(1024) void k_row_sum(const float* in, long rows, long cols, const RowSumOut out) {
  __shared__ double s[16][64];
  const long c = (long)blockIdx.x * 64 + threadIdx.x;
  double v = 0.0;
  if (c < cols)
    for (long r = threadIdx.y; r < rows; r += 16) v += in[r * cols + c];
  s[threadIdx.y][threadIdx.x] = v;
  __syncthreads();
  if (threadIdx.y || c >= cols) return;
  v = 0.0;
#pragma unroll
  for (int k = 0; k < 16; ++k) v += s[k][threadIdx.x];
  for (int i = 0; i < 3; ++i) {
    if (c < out.begin[i] || c >= out.begin[i + 1] || !out.ptr[i]) continue;
    const long q = c - out.begin[i];
    store_as(out.ptr[i], out.type[i], (q % out.minor[i]) * out.major[i] + q / out.minor[i], (float)v);
  }
}

template <class T, int W>
int launch(int what, const ConvArgs& a, long groups, hipStream_t st) {
  if (what == 0) hipLaunchKernelGGL((k_conv<T, W>), dim3((unsigned)groups), dim3(256), 0, st, a);
  else if (what == 1) hipLaunchKernelGGL((k_conv_grad<T, W>), dim3((unsigned)groups), dim3(256), 0, st, a);
  else hipLaunchKernelGGL((k_conv_step<T, W>), dim3((unsigned)groups), dim3(256), 0, st, a);
  return (int)last();
}

template <class T>
int by_width(int what, const ConvArgs& a, long groups, hipStream_t st) {
  switch (a.p.W) {
    case 1: return launch<T, 1>(what, a, groups, st);
    case 2: return launch<T, 2>(what, a, groups, st);
    case 3: return launch<T, 3>(what, a, groups, st);
    case 4: return launch<T, 4>(what, a, groups, st);
    case 5: return launch<T, 5>(what, a, groups, st);
    case 6: return launch<T, 6>(what, a, groups, st);
    case 7: return launch<T, 7>(what, a, groups, st);
    default: return launch<T, 8>(what, a, groups, st);
  }
}

int by_type(int what, const ConvArgs& a, long groups, hipStream_t st) {
  if (!grid_fits(groups, 256)) return LQG_ERR_ARG;
  if (a.p.type == LQG_T_F32) return by_width<float>(what, a, groups, st);
  if (a.p.type == LQG_T_BF16) return by_width<bf16>(what, a, groups, st);
  return by_width<f16>(what, a, groups, st);
}

int check(const lqg_conv* p, bool step) {
  if (!p) return LQG_ERR_NULL;
  if (p->W < 1 || p->W > WMAX || p->B < 1 || p->T < 1 || p->D < 1 || (step && p->T != 1)) return LQG_ERR_ARG;
  if (p->type != LQG_T_F32 && p->type != LQG_T_BF16 && p->type != LQG_T_F16) return LQG_ERR_ARG;
  for (const lqg_param* q : {&p->w, &p->bias})
    if (q->ptr && q->type != LQG_T_F32 && q->type != LQG_T_BF16 && q->type != LQG_T_F16) return LQG_ERR_ARG;
  if (!p->x.ptr || !p->w.ptr || (step && p->W > 1 && !p->state)) return LQG_ERR_NULL;
  return 0;
}

}  // namespace

namespace lqg {
namespace learn {
hipError_t row_sum(const RowSum& s, const RowSumOut& out, hipStream_t stream) {
  const long blocks = (s.cols + 63) / 64;
  const float* in = s.in;
  long rows = s.rows;
  if (const long mid = row_sum_mid_rows(rows)) {
    hipLaunchKernelGGL(k_row_sum_mid, dim3((unsigned)(blocks * mid)), dim3(64, 16), 0, stream, in, rows, s.cols, mid, s.mid);
    in = s.mid;
    rows = mid;
  }
  hipLaunchKernelGGL(k_row_sum, dim3((unsigned)blocks), dim3(64, 16), 0, stream, in, rows, s.cols, out);
  return hipGetLastError();
}
}  // namespace learn
}  // namespace lqg

extern "C" int lqg_causal_conv(const lqg_conv* p, void* stream) {
  if (const int rc = check(p, false)) return rc;
  if (!p->y.ptr) return LQG_ERR_NULL;
  ConvArgs a{};
  a.p = *p;
  a.pieces = (p->T + PIECE - 1) / PIECE;
  a.blocks = (p->D + 255) / 256;
  return by_type(0, a, a.blocks * a.pieces * p->B, (hipStream_t)stream);
}

extern "C" size_t lqg_causal_conv_grad_workspace(const lqg_conv* p) {
  if (check(p, false)) return 0;
  const long rows = p->B * ((p->T + GPIECE - 1) / GPIECE), cols = (p->W + 1) * p->D;
  return (size_t)(rows + row_sum_mid_rows(rows)) * cols * sizeof(float);
}

extern "C" int lqg_causal_conv_grad(const lqg_conv* p, lqg_seq dy, const void* dstate_out, void* dx, void* dstate, void* dw,
                                    void* dbias, void* workspace, size_t workspace_bytes, void* stream) {
  if (const int rc = check(p, false)) return rc;
  if (!dy.ptr || !dx || !workspace) return LQG_ERR_NULL;
  if (workspace_bytes < lqg_causal_conv_grad_workspace(p)) return LQG_ERR_WORKSPACE;
  ConvArgs a{};
  a.p = *p;
  a.pieces = (p->T + GPIECE - 1) / GPIECE;
  a.blocks = (p->D + 255) / 256;
  a.dy = dy;
  a.dstate_out = dstate_out;
  a.dx = dx;
  a.dstate = dstate;
  a.part = static_cast<float*>(workspace);
  if (const int rc = by_type(1, a, a.blocks * a.pieces * p->B, (hipStream_t)stream)) return rc;
  if (!dw && !dbias) return 0;
  const long rows = p->B * a.pieces, cols = (p->W + 1) * p->D;
  RowSum s{a.part, rows, cols, a.part + rows * cols};
  RowSumOut o{};
  o.ptr[0] = dw;
  o.type[0] = p->w.type;
  o.major[0] = p->W;
  o.minor[0] = p->D;
  o.ptr[1] = dbias;
  o.type[1] = p->bias.type;
  o.major[1] = 1;
  o.minor[1] = p->D;
  o.begin[1] = p->W * p->D;
  o.begin[2] = o.begin[3] = cols;
  o.major[2] = o.minor[2] = 1;
  return (int)row_sum(s, o, (hipStream_t)stream);
}

extern "C" int lqg_causal_conv_step(const lqg_conv* p, void* stream) {
  if (const int rc = check(p, true)) return rc;
  if (!p->y.ptr) return LQG_ERR_NULL;
  ConvArgs a{};
  a.p = *p;
  a.blocks = (p->D + 255) / 256;
  return by_type(2, a, a.blocks * p->B, (hipStream_t)stream);
}
