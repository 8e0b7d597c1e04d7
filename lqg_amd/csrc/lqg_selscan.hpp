// lqg_selscan.hpp — kernels of the selective state-space scan: forward, gradients, single step (include/lqg_learn.h).
//
//   dl = softplus(delta + delta_bias),  h_t = exp(dl_t A) h_{t-1} + dl_t B_t u_t,  y_t = (sum_n C_t h_t + D u_t) silu(z_t)
//
// B x D x N scalar recurrences; per step of one of them one exponential and four float operations, and B_t, C_t are shared by all
// channels of a group.  Mapping: a lane is a channel, a wave holds NS of the N states of 64 channels in registers, the NW = N / NS
// waves of a workgroup share those 64 channels.  The time axis is walked in tiles of TT steps: each wave prepares TT / NW rows
// (softplus, dl u) for all of them through LDS, runs the tile's TT steps on its states, and leaves its part of sum_n C h in LDS, where
// the waves finish TT / NW rows each.  B_t and C_t of a tile sit one value per lane in rows of 16 and reach the arithmetic as DPP row
// broadcasts: an operand modifier, no load and no instruction.  Few channels: the time axis is cut into chunks; one pass leaves each
// chunk's end state from zero and its sum of dl, the second enters with exp(A sum dl) h + end state over the chunks before it.
#pragma once
#include "lqg_learn.hpp"

namespace lqg {
namespace learn {

constexpr float LN2 = 0.6931471805599453f;

struct ScanArgs {
  lqg_selscan p;
  lqg_selscan_bars g;
  long Dg, bpg, blocks;          // channels of a group, blocks of 64 of them, blocks in all
  long chunks, chunk, tiles;     // chunks of the time axis, their steps (a multiple of TT), tiles of TT steps in T
  float *hl, *sd;                // carries [B][chunks][N][D], sums of dl [B][chunks][D]
  float *partB, *partC, *partP;  // gradients: [blocks][B][T][N] twice, [B * chunks][N + 2][D]
};

template <class IT> __device__ inline const IT* seq(const lqg_seq& s, long b, long off) {
  return static_cast<const IT*>(s.ptr) + b * s.sb + off;
}

// where a workgroup is
template <int NS, int TT> struct Place {
  int lane, w;
  long blk, b, c, grp, d, n0, len, t0, t1, tiles;
  bool on;
  __device__ Place(const ScanArgs& a) {
    lane = threadIdx.x;
    w = __builtin_amdgcn_readfirstlane((int)threadIdx.y);
    blk = blockIdx.x % a.blocks;
    const long rest = blockIdx.x / a.blocks;
    c = rest % a.chunks;
    b = rest / a.chunks;
    grp = blk / a.bpg;
    const long in = (blk % a.bpg) * 64 + lane;
    on = in < a.Dg;
    d = grp * a.Dg + (on ? in : a.Dg - 1);          // lanes past the group's end repeat its last channel and store nothing
    n0 = w * NS;
    len = a.p.T;
    if (a.p.lengths) {
      const long l = a.p.lengths[b];
      len = l < 0 ? 0 : (l < len ? l : len);
    }
    t0 = c * a.chunk;
    t1 = min(t0 + a.chunk, a.p.T);
    const long end = min(t1, len);
    tiles = end > t0 ? (end - t0 + TT - 1) / TT : 0;
  }
};

template <int NS> __device__ inline void load_A2(const ScanArgs& a, long d, long n0, float (&A2)[NS]) {
#pragma unroll
  for (int j = 0; j < NS; ++j) A2[j] = n0 + j < a.p.N ? load_param(a.p.A, d * a.p.N + n0 + j) * LOG2E : 0.0f;
}

// a tile's B or C: value (t, j) in register (t NS + j) / 16, lane (t NS + j) % 16 of each row; 0 behind the end and past N
template <class IT, int NS, int TT>
__device__ inline void load_bc(const lqg_seq& s, long b, long grp, long t0, long n0, long len, long N, int lane, float (&r)[TT * NS / 16]) {
#pragma unroll
  for (int q = 0; q < TT * NS / 16; ++q) {
    const int f = q * 16 + (lane & 15);
    const long t = t0 + f / NS, n = n0 + f % NS;
    r[q] = t < len && n < N ? up(seq<IT>(s, b, grp * s.sg)[t * s.st + n]) : 0.0f;
  }
}
template <int NS, int T, int J, int Q> __device__ inline float bc(const float (&r)[Q]) {
  return row_bcast<(T * NS + J) % 16>(r[(T * NS + J) / 16]);
}

// compile-time loop: f(integral_constant<int, I>) for I = 0 .. N-1
template <int I> struct Int { static constexpr int v = I; };
template <int N, int I = 0, class F> __device__ __forceinline__ void each(F&& f) {
  if constexpr (I < N) {
    f(Int<I>{});
    each<N, I + 1>(f);
  }
}
template <int I, class F> __device__ __forceinline__ void each_back(F&& f) {
  if constexpr (I >= 0) {
    f(Int<I>{});
    each_back<I - 1>(f);
  }
}

__device__ inline float step_size(const ScanArgs& a, float raw) { return a.p.softplus ? softplus(raw) : raw; }

// ------------------------------------------------------------------------------------------------ forward
// CARRY: leave each chunk's end state from zero and its sum of dl instead of y.
template <class IT, int NS, int NW, int TT, bool CARRY>
__global__ __launch_bounds__(64 * NW) void k_scan(const ScanArgs a) {
  constexpr int RW = TT / NW, Q = TT * NS / 16;
  __shared__ float2 s_in[2][TT][64];
  __shared__ float s_y[CARRY ? 1 : 2][CARRY ? 1 : TT][NW][64];
  const Place<NS, TT> at(a);
  const long D = a.p.D, N = a.p.N, d = at.d, b = at.b;
  const int lane = at.lane, w = at.w;
  float A2[NS], h[NS], sum = 0.0f;
  load_A2<NS>(a, d, at.n0, A2);
#pragma unroll
  for (int j = 0; j < NS; ++j)
    h[j] = !CARRY && a.p.state && at.n0 + j < N ? a.p.state[(b * D + d) * N + at.n0 + j] : 0.0f;
  if (!CARRY) {
    for (long c = 0; c < at.c; ++c) {                   // the chunks before this one
      const float sd = a.sd[(b * a.chunks + c) * D + d];
      const float* hl = a.hl + ((b * a.chunks + c) * N + at.n0) * D + d;
#pragma unroll
      for (int j = 0; j < NS; ++j)
        if (at.n0 + j < N) h[j] = fmaf(exp2_hw(sd * A2[j]), h[j], hl[j * D]);
    }
  }
  const float bias = a.p.delta_bias.ptr ? load_param(a.p.delta_bias, d) : 0.0f;
  const float Dk = !CARRY && a.p.Dskip.ptr ? load_param(a.p.Dskip, d) : 0.0f;
  const bool gate = !CARRY && a.p.z.ptr;
  struct Rows { IT u[RW], dl[RW], z[RW]; };
  auto load = [&](Rows& r, long t0) {
#pragma unroll
    for (int i = 0; i < RW; ++i) {
      const long t = min(t0 + w * RW + i, at.len - 1);
      r.u[i] = seq<IT>(a.p.u, b, t * a.p.u.st)[d];
      r.dl[i] = seq<IT>(a.p.delta, b, t * a.p.delta.st)[d];
      if (gate) r.z[i] = seq<IT>(a.p.z, b, t * a.p.z.st)[d];
    }
  };
  auto prepare = [&](const Rows& r, long t0, int buf) {
#pragma unroll
    for (int i = 0; i < RW; ++i) {
      const bool live = t0 + w * RW + i < at.len;
      const float dl = live ? step_size(a, up(r.dl[i]) + bias) : 0.0f;
      s_in[buf][w * RW + i][lane] = make_float2(dl, live ? dl * up(r.u[i]) : 0.0f);
    }
  };
  IT* y = CARRY ? nullptr : const_cast<IT*>(seq<IT>(a.p.y, b, d));
  auto finish = [&](const Rows& r, long t0, int buf) {
#pragma unroll
    for (int i = 0; i < RW; ++i) {
      const long t = t0 + w * RW + i;
      float v = 0.0f;
#pragma unroll
      for (int k = 0; k < NW; ++k) v += s_y[buf][w * RW + i][k][lane];
      v = fmaf(Dk, up(r.u[i]), v);
      if (gate) {
        const float z = up(r.z[i]);
        v *= z * sigmoid(z);
      }
      if (t < at.t1 && at.on) y[t * a.p.y.st] = down<IT>(t < at.len ? v : 0.0f);
    }
  };

  Rows before, now, next, after;
  float B[Q], C[Q], Bn[Q], Cn[Q];
  if (at.tiles > 0) {
    load(now, at.t0);
    load_bc<IT, NS, TT>(a.p.Bm, b, at.grp, at.t0, at.n0, at.len, N, lane, B);
    if (!CARRY) load_bc<IT, NS, TT>(a.p.Cm, b, at.grp, at.t0, at.n0, at.len, N, lane, C);
    prepare(now, at.t0, 0);
    if (at.tiles > 1) load(next, at.t0 + TT);
  }
  __syncthreads();
  for (long i = 0; i < at.tiles; ++i) {
    const long t0 = at.t0 + i * TT;
    const int buf = (int)(i & 1);
    if (i + 1 < at.tiles) {
      prepare(next, t0 + TT, buf ^ 1);
      load_bc<IT, NS, TT>(a.p.Bm, b, at.grp, t0 + TT, at.n0, at.len, N, lane, Bn);
      if (!CARRY) load_bc<IT, NS, TT>(a.p.Cm, b, at.grp, t0 + TT, at.n0, at.len, N, lane, Cn);
    }
    if (i + 2 < at.tiles) load(after, t0 + 2 * TT);
    if (!CARRY && a.p.checkpoints && at.on) {
      float* ck = static_cast<float*>(a.p.checkpoints) + ((b * a.tiles + t0 / TT) * N + at.n0) * D + d;
#pragma unroll
      for (int j = 0; j < NS; ++j)
        if (at.n0 + j < N) ck[j * D] = h[j];
    }
    each<TT>([&](auto tc) {
      constexpr int t = decltype(tc)::v;
      const float2 in = s_in[buf][t][lane];
      float v = 0.0f;
      each<NS>([&](auto jc) {
        constexpr int j = decltype(jc)::v;
        h[j] = fmaf(exp2_hw(in.x * A2[j]), h[j], bc<NS, t, j>(B) * in.y);
        if (!CARRY) v = fmaf(bc<NS, t, j>(C), h[j], v);
      });
      if (CARRY) sum += in.x;
      else s_y[buf][t][w][lane] = v;
    });
    if (!CARRY && i > 0) finish(before, t0 - TT, buf ^ 1);
    before = now;
    now = next;
    next = after;
#pragma unroll
    for (int q = 0; q < Q; ++q) B[q] = Bn[q], C[q] = Cn[q];
    __syncthreads();
  }
  if (CARRY) {
    if (!at.on) return;
    float* hl = a.hl + ((b * a.chunks + at.c) * N + at.n0) * D + d;
#pragma unroll
    for (int j = 0; j < NS; ++j)
      if (at.n0 + j < N) hl[j * D] = h[j];
    if (w == 0) a.sd[(b * a.chunks + at.c) * D + d] = sum;
    return;
  }
  if (at.tiles > 0) finish(before, at.t0 + (at.tiles - 1) * TT, (int)((at.tiles - 1) & 1));
  if (!at.on) return;
  for (long t = at.t0 + at.tiles * TT + w; t < at.t1; t += NW) y[t * a.p.y.st] = down<IT>(0.0f);
  if (a.p.state_out && at.c == a.chunks - 1) {
#pragma unroll
    for (int j = 0; j < NS; ++j)
      if (at.n0 + j < N) a.p.state_out[(b * D + d) * N + at.n0 + j] = h[j];
  }
}

// ------------------------------------------------------------------------------------------------ gradients
// With dY = dy silu(z) and lambda the carry from the future (lambda = a_{t+1} g_{t+1}):
//   g = C dY + lambda;  dC = sum_d dY h;  dB = sum_d g dl u;  s1 = sum_n g B;  q = g a h_{t-1};  s2 = sum_n A q;
//   du = dl s1 + D dY;  d dl = s2 + u s1;  dA = sum q dl;  lambda <- a g.
// A tile's states are recomputed from the checkpoint that the forward pass left at its start.

// x and y reduced by halves: lanes whose bit BIT is 0 receive x's sum over that bit, the others y's.
template <int BIT> __device__ inline float merge(float x, float y, int lane) {
  if constexpr (BIT == 5) {
    const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(y), false, false);
    return __uint_as_float(r[0]) + __uint_as_float(r[1]);
  } else if constexpr (BIT == 4) {
    const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(y), false, false);
    return __uint_as_float(r[0]) + __uint_as_float(r[1]);
  } else {
    const bool hi = lane >> BIT & 1;
    const float keep = hi ? y : x, give = hi ? x : y;
    return keep + dpp<BIT == 3 ? DPP_ROR8 : BIT == 2 ? DPP_HALF_MIRROR : BIT == 1 ? DPP_XOR2 : DPP_XOR1>(give);
  }
}

// CARRY: leave each chunk's carry (lambda at its start from 0 at its end) and its sum of dl.
template <class IT, int NS, int NW, int TT, bool CARRY>
__global__ __launch_bounds__(64 * NW) void k_scan_grad(const ScanArgs a) {
  constexpr int RW = TT / NW, Q = TT * NS / 16;
  __shared__ float2 s_in[2][TT][64];
  __shared__ float s_dy[2][TT][64];
  __shared__ float2 s_sum[CARRY ? 1 : TT][NW][64];
  __shared__ float s_y[CARRY ? 1 : TT][NW][64];
  const Place<NS, TT> at(a);
  const long D = a.p.D, N = a.p.N, T = a.p.T, d = at.d, b = at.b;
  const int lane = at.lane, w = at.w;
  float A2[NS], lam[NS], dA[NS], sum = 0.0f, dDk = 0.0f, dbias = 0.0f;
  load_A2<NS>(a, d, at.n0, A2);
#pragma unroll
  for (int j = 0; j < NS; ++j) {
    dA[j] = 0.0f;
    lam[j] = !CARRY && a.g.dstate_out && at.n0 + j < N ? a.g.dstate_out[(b * D + d) * N + at.n0 + j] : 0.0f;
  }
  if (!CARRY) {
    for (long c = a.chunks - 1; c > at.c; --c) {        // the chunks after this one
      const float sd = a.sd[(b * a.chunks + c) * D + d];
      const float* hl = a.hl + ((b * a.chunks + c) * N + at.n0) * D + d;
#pragma unroll
      for (int j = 0; j < NS; ++j)
        if (at.n0 + j < N) lam[j] = fmaf(exp2_hw(sd * A2[j]), lam[j], hl[j * D]);
    }
  }
  const float bias = a.p.delta_bias.ptr ? load_param(a.p.delta_bias, d) : 0.0f;
  const float Dk = a.p.Dskip.ptr ? load_param(a.p.Dskip, d) : 0.0f;
  const bool gate = a.p.z.ptr;
  struct Rows { IT u[RW], dl[RW], z[RW], dy[RW]; };
  auto load = [&](Rows& r, long t0) {
#pragma unroll
    for (int i = 0; i < RW; ++i) {
      const long t = min(t0 + w * RW + i, at.len - 1);
      r.u[i] = seq<IT>(a.p.u, b, t * a.p.u.st)[d];
      r.dl[i] = seq<IT>(a.p.delta, b, t * a.p.delta.st)[d];
      r.dy[i] = seq<IT>(a.g.dy, b, t * a.g.dy.st)[d];
      if (gate) r.z[i] = seq<IT>(a.p.z, b, t * a.p.z.st)[d];
    }
  };
  auto prepare = [&](const Rows& r, long t0, int buf) {
#pragma unroll
    for (int i = 0; i < RW; ++i) {
      const bool live = t0 + w * RW + i < at.len && at.on;
      const float dl = live ? step_size(a, up(r.dl[i]) + bias) : 0.0f;
      float dy = up(r.dy[i]);
      if (gate) {
        const float z = up(r.z[i]);
        dy *= z * sigmoid(z);
      }
      s_in[buf][w * RW + i][lane] = make_float2(dl, live ? dl * up(r.u[i]) : 0.0f);
      s_dy[buf][w * RW + i][lane] = live ? dy : 0.0f;
    }
  };
  const long out0 = b * T * D + d;
  auto finish = [&](const Rows& r, long t0, int buf) {
#pragma unroll
    for (int i = 0; i < RW; ++i) {
      const int row = w * RW + i;
      const long t = t0 + row;
      float s1 = 0.0f, s2 = 0.0f;
#pragma unroll
      for (int k = 0; k < NW; ++k) {
        const float2 s = s_sum[row][k][lane];
        s1 += s.x;
        s2 += s.y;
      }
      const float dl = s_in[buf][row][lane].x, dY = s_dy[buf][row][lane], u = up(r.u[i]);
      const bool live = t < at.len;
      float ddl = fmaf(u, s1, LN2 * s2);
      if (a.p.softplus) ddl *= sigmoid(up(r.dl[i]) + bias);
      if (live && at.on) {
        dDk = fmaf(dY, u, dDk);
        dbias += ddl;
      }
      if (t < at.t1 && at.on) {
        static_cast<IT*>(a.g.du)[out0 + t * D] = down<IT>(live ? fmaf(dl, s1, Dk * dY) : 0.0f);
        static_cast<IT*>(a.g.ddelta)[out0 + t * D] = down<IT>(live ? ddl : 0.0f);
      }
      if (gate) {
        float y = Dk * u;
#pragma unroll
        for (int k = 0; k < NW; ++k) y += s_y[row][k][lane];
        const float z = up(r.z[i]), sg = sigmoid(z);
        const float dz = up(r.dy[i]) * y * (sg * fmaf(z, 1.0f - sg, 1.0f));
        if (t < at.t1 && at.on) static_cast<IT*>(a.g.dz)[out0 + t * D] = down<IT>(live ? dz : 0.0f);
      }
    }
  };

  const float* ck = CARRY ? nullptr : static_cast<const float*>(a.p.checkpoints) + (b * a.tiles * N + at.n0) * D + d;
  Rows now, next;
  float B[Q], C[Q], h0[NS];
  auto load_tile = [&](long t0) {
    load_bc<IT, NS, TT>(a.p.Cm, b, at.grp, t0, at.n0, at.len, N, lane, C);
    if (CARRY) return;
    load_bc<IT, NS, TT>(a.p.Bm, b, at.grp, t0, at.n0, at.len, N, lane, B);
#pragma unroll
    for (int j = 0; j < NS; ++j) h0[j] = at.n0 + j < N ? ck[((t0 / TT) * N + j) * D] : 0.0f;
  };
  if (at.tiles > 0) {
    load(now, at.t0 + (at.tiles - 1) * TT);
    prepare(now, at.t0 + (at.tiles - 1) * TT, (int)((at.tiles - 1) & 1));
  }
  __syncthreads();
  for (long i = at.tiles - 1; i >= 0; --i) {
    const long t0 = at.t0 + i * TT;
    const int buf = (int)(i & 1);
    load_tile(t0);
    if (i > 0) load(next, t0 - TT);
    if constexpr (CARRY) {
      each_back<TT - 1>([&](auto tc) {
        constexpr int t = decltype(tc)::v;
        const float dl = s_in[buf][t][lane].x, dY = s_dy[buf][t][lane];
        sum += dl;
        each<NS>([&](auto jc) {
          constexpr int j = decltype(jc)::v;
          lam[j] = exp2_hw(dl * A2[j]) * fmaf(bc<NS, t, j>(C), dY, lam[j]);
        });
      });
    } else {
      float hh[TT][NS], aa[TT][NS];
      each<TT>([&](auto tc) {
        constexpr int t = decltype(tc)::v;
        const float2 in = s_in[buf][t][lane];
        float y = 0.0f;
        each<NS>([&](auto jc) {
          constexpr int j = decltype(jc)::v;
          aa[t][j] = exp2_hw(in.x * A2[j]);
          hh[t][j] = fmaf(aa[t][j], t ? hh[t ? t - 1 : 0][j] : h0[j], bc<NS, t, j>(B) * in.y);
          if (gate) y = fmaf(bc<NS, t, j>(C), hh[t][j], y);
        });
        if (gate) s_y[t][w][lane] = y;
      });
      float tA[NS];
#pragma unroll
      for (int j = 0; j < NS; ++j) tA[j] = 0.0f;
      // dB, dC of 8 steps x 8 values end as one value per lane: step bits on lane bits 5, 4, 3, value bits on 2, 1, 0
      constexpr int K = 2 * NS;
      float p0[K], p1[K], p2[K];
      each_back<TT - 1>([&](auto tc) {
        constexpr int t = decltype(tc)::v;
        const float2 in = s_in[buf][t][lane];
        const float dY = s_dy[buf][t][lane];
        float v[K], s1 = 0.0f, s2 = 0.0f;
        each<NS>([&](auto jc) {
          constexpr int j = decltype(jc)::v;
          const float g = fmaf(bc<NS, t, j>(C), dY, lam[j]);
          v[j] = g * in.y;
          v[NS + j] = dY * hh[t][j];
          s1 = fmaf(bc<NS, t, j>(B), g, s1);
          lam[j] = aa[t][j] * g;
          const float q = lam[j] * (t ? hh[t ? t - 1 : 0][j] : h0[j]);
          s2 = fmaf(A2[j], q, s2);
          tA[j] = fmaf(q, in.x, tA[j]);
        });
        s_sum[t][w][lane] = make_float2(s1, s2);
        if constexpr (t & 1) {
#pragma unroll
          for (int k = 0; k < K; ++k) p0[k] = v[k];
        } else {
#pragma unroll
          for (int k = 0; k < K; ++k) v[k] = merge<5>(v[k], p0[k], lane);
          if constexpr (t & 2) {
#pragma unroll
            for (int k = 0; k < K; ++k) p1[k] = v[k];
          } else {
#pragma unroll
            for (int k = 0; k < K; ++k) v[k] = merge<4>(v[k], p1[k], lane);
            if constexpr (t & 4) {
#pragma unroll
              for (int k = 0; k < K; ++k) p2[k] = v[k];
            } else {
#pragma unroll
              for (int k = 0; k < K; ++k) v[k] = merge<3>(v[k], p2[k], lane);
#pragma unroll
              for (int o = 0; o < K; o += 8) {
                float x[4];
#pragma unroll
                for (int k = 0; k < 4; ++k) x[k] = merge<2>(v[o + k], v[o + k + 4], lane);
                x[0] = merge<1>(x[0], x[2], lane);
                x[1] = merge<1>(x[1], x[3], lane);
                x[0] = merge<0>(x[0], x[1], lane);
                const int k = o + (lane & 4) + (lane & 1) * 1 + (lane & 2);
                const long ts = t0 + t + (lane >> 5 & 1) + (lane >> 4 & 1) * 2 + (lane >> 3 & 1) * 4;
                const long n = at.n0 + k % NS;
                float* part = k < NS ? a.partB : a.partC;
                if (ts < at.t1 && n < N) part[((at.blk * a.p.B + b) * T + ts) * N + n] = x[0];
              }
            }
          }
        }
      });
#pragma unroll
      for (int j = 0; j < NS; ++j) dA[j] += tA[j];
    }
    if constexpr (CARRY) {
      if (i > 0) prepare(next, t0 - TT, buf ^ 1);
      __syncthreads();
    } else {
      __syncthreads();
      finish(now, t0, buf);
      if (i > 0) prepare(next, t0 - TT, buf ^ 1);
      now = next;
      __syncthreads();
    }
  }
  if constexpr (CARRY) {
    if (!at.on) return;
    float* hl = a.hl + ((b * a.chunks + at.c) * N + at.n0) * D + d;
#pragma unroll
    for (int j = 0; j < NS; ++j)
      if (at.n0 + j < N) hl[j * D] = lam[j];
    if (w == 0) a.sd[(b * a.chunks + at.c) * D + d] = sum;
  } else {
    for (long t = at.t0 + at.tiles * TT + w; t < at.t1; t += NW) {       // padding
      if (!at.on) break;
      static_cast<IT*>(a.g.du)[out0 + t * D] = down<IT>(0.0f);
      static_cast<IT*>(a.g.ddelta)[out0 + t * D] = down<IT>(0.0f);
      if (gate) static_cast<IT*>(a.g.dz)[out0 + t * D] = down<IT>(0.0f);
    }
    s_sum[0][w][lane] = make_float2(dDk, dbias);
    __syncthreads();
    if (!at.on) return;
    float* part = a.partP + (b * a.chunks + at.c) * (N + 2) * D + d;
#pragma unroll
    for (int j = 0; j < NS; ++j)
      if (at.n0 + j < N) {
        part[(at.n0 + j) * D] = dA[j];
        if (a.g.dstate && at.c == 0) a.g.dstate[(b * D + d) * N + at.n0 + j] = lam[j];
      }
    if (w == 0) {
      float2 s = make_float2(0.0f, 0.0f);
#pragma unroll
      for (int k = 0; k < NW; ++k) s.x += s_sum[0][k][lane].x, s.y += s_sum[0][k][lane].y;
      part[N * D] = s.x;
      part[(N + 1) * D] = s.y;
    }
  }
}

// dB, dC [B][T][G][N]: the blocks of a group summed, 0 in the padding
template <class IT> __global__ __launch_bounds__(256) void k_scan_groups(const ScanArgs a) {
  const long e = (long)blockIdx.x * 256 + threadIdx.x, N = a.p.N, G = a.p.G, T = a.p.T, B = a.p.B;
  if (e >= B * T * G * N) return;
  const long n = e % N, g = e / N % G, t = e / (N * G) % T, b = e / (N * G * T);
  const bool live = !a.p.lengths || t < a.p.lengths[b];
  float x = 0.0f, y = 0.0f;
  if (live)
    for (long k = g * a.bpg; k < (g + 1) * a.bpg; ++k) {
      const long at = ((k * B + b) * T + t) * N + n;
      x += a.partB[at];
      y += a.partC[at];
    }
  static_cast<IT*>(a.g.dBm)[e] = down<IT>(x);
  static_cast<IT*>(a.g.dCm)[e] = down<IT>(y);
}

// ------------------------------------------------------------------------------------------------ one step
// LPC lanes per channel, 4 states each: a wave moves whole lines of the state.
template <class IT, int LPC>
__global__ __launch_bounds__(256) void k_scan_step(const ScanArgs a, float* state) {
  const long N = a.p.N, D = a.p.D, per = 256 / LPC;
  const long blk = blockIdx.x % a.blocks, b = blockIdx.x / a.blocks;
  const long d = blk * per + threadIdx.x / LPC;
  const int q = threadIdx.x % LPC;
  if (d >= D) return;                                 // whole channels: their LPC lanes leave together
  const long grp = d / a.Dg;
  const float u = up(seq<IT>(a.p.u, b, d)[0]);
  float dl = up(seq<IT>(a.p.delta, b, d)[0]);
  if (a.p.delta_bias.ptr) dl += load_param(a.p.delta_bias, d);
  dl = step_size(a, dl);
  const IT* B = seq<IT>(a.p.Bm, b, grp * a.p.Bm.sg);
  const IT* C = seq<IT>(a.p.Cm, b, grp * a.p.Cm.sg);
  float* h = state + (b * D + d) * N;
  float y = 0.0f;
  for (long n = q * 4; n < N; n += LPC * 4) {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      if (n + j >= N) break;
      const float v = fmaf(exp2_hw(dl * (load_param(a.p.A, d * N + n + j) * LOG2E)), h[n + j], dl * u * up(B[n + j]));
      h[n + j] = v;
      y = fmaf(up(C[n + j]), v, y);
    }
  }
#pragma unroll
  for (int k = 1; k < LPC; k <<= 1) y += __shfl_xor(y, k);
  if (q) return;
  if (a.p.Dskip.ptr) y = fmaf(load_param(a.p.Dskip, d), u, y);
  if (a.p.z.ptr) {
    const float z = up(seq<IT>(a.p.z, b, d)[0]);
    y *= z * sigmoid(z);
  }
  const_cast<IT*>(seq<IT>(a.p.y, b, d))[0] = down<IT>(y);
}

// ------------------------------------------------------------------------------------------------ launches
inline int waves_of(long N) { return N > 16 ? 8 : N > 8 ? 4 : N > 4 ? 2 : 1; }

template <class IT, int NS, int NW, int TT> int launch(int what, const ScanArgs& a, hipStream_t st) {
  const long groups = a.blocks * a.chunks * a.p.B;
  if (!grid_fits(groups, 64 * NW)) return LQG_ERR_ARG;
  const dim3 g((unsigned)groups), t(64, NW);
  if (what == 0) {
    if (a.chunks > 1) hipLaunchKernelGGL((k_scan<IT, NS, NW, TT, true>), g, t, 0, st, a);
    hipLaunchKernelGGL((k_scan<IT, NS, NW, TT, false>), g, t, 0, st, a);
  } else {
    if (a.chunks > 1) hipLaunchKernelGGL((k_scan_grad<IT, NS, NW, TT, true>), g, t, 0, st, a);
    hipLaunchKernelGGL((k_scan_grad<IT, NS, NW, TT, false>), g, t, 0, st, a);
  }
  return (int)last();
}

template <class IT> int by_states(int what, const ScanArgs& a, hipStream_t st) {
  if (a.p.N > 32) return launch<IT, 8, 8, 8>(what, a, st);
  switch (waves_of(a.p.N)) {
    case 1: return launch<IT, 4, 1, 16>(what, a, st);
    case 2: return launch<IT, 4, 2, 16>(what, a, st);
    case 4: return launch<IT, 4, 4, 16>(what, a, st);
    default: return launch<IT, 4, 8, 16>(what, a, st);
  }
}
template <class IT> int launch_step(ScanArgs a, float* state, hipStream_t st) {
  const int lpc = a.p.N > 32 ? 16 : a.p.N > 16 ? 8 : a.p.N > 8 ? 4 : a.p.N > 4 ? 2 : 1;
  a.blocks = (a.p.D * lpc + 255) / 256;
  const long groups = a.blocks * a.p.B;
  if (!grid_fits(groups, 256)) return LQG_ERR_ARG;
  const dim3 g((unsigned)groups), t(256);
  switch (lpc) {
    case 1: hipLaunchKernelGGL((k_scan_step<IT, 1>), g, t, 0, st, a, state); break;
    case 2: hipLaunchKernelGGL((k_scan_step<IT, 2>), g, t, 0, st, a, state); break;
    case 4: hipLaunchKernelGGL((k_scan_step<IT, 4>), g, t, 0, st, a, state); break;
    case 8: hipLaunchKernelGGL((k_scan_step<IT, 8>), g, t, 0, st, a, state); break;
    default: hipLaunchKernelGGL((k_scan_step<IT, 16>), g, t, 0, st, a, state); break;
  }
  return (int)last();
}

template <class IT> int launch_groups(const ScanArgs& a, long groups, hipStream_t st) {
  hipLaunchKernelGGL(k_scan_groups<IT>, dim3((unsigned)groups), dim3(256), 0, st, a);
  return (int)last();
}

// what: 0 forward, 1 gradients; each type of sequence is a translation unit of its own
template <class IT> struct ScanOf {
  static int run(int what, const ScanArgs& a, hipStream_t st);
  static int groups(const ScanArgs& a, long groups, hipStream_t st);
  static int step(const ScanArgs& a, float* state, hipStream_t st);
};

}  // namespace learn
}  // namespace lqg
