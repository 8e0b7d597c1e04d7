// lqg_selscan.hip — selective state-space scan (include/lqg_learn.h): with -DLQG_SELSCAN_TYPE=<type> the kernels for sequences of that
// type, without it the C entry points.
#include "lqg_selscan.hpp"

#include <algorithm>
#include <cmath>

using namespace lqg::learn;

#ifdef LQG_SELSCAN_TYPE
namespace lqg {
namespace learn {
typedef LQG_SELSCAN_TYPE IT;
template <> int ScanOf<IT>::run(int what, const ScanArgs& a, hipStream_t st) { return by_states<IT>(what, a, st); }
template <> int ScanOf<IT>::groups(const ScanArgs& a, long groups, hipStream_t st) { return launch_groups<IT>(a, groups, st); }
template <> int ScanOf<IT>::step(const ScanArgs& a, float* state, hipStream_t st) { return launch_step<IT>(a, state, st); }
}  // namespace learn
}  // namespace lqg
#else
namespace lqg {
namespace learn {
#define X(IT)                                                                         \
  template <> int ScanOf<IT>::run(int, const ScanArgs&, hipStream_t);                 \
  template <> int ScanOf<IT>::groups(const ScanArgs&, long, hipStream_t);             \
  template <> int ScanOf<IT>::step(const ScanArgs&, float*, hipStream_t);
X(float) X(bf16) X(f16)
#undef X
}  // namespace learn
}  // namespace lqg

namespace {

constexpr int64_t MAX_STRIDE = (1 << 22) - 1;  // rows of a tile are at 32-bit byte offsets, products of 24-bit numbers

int check(const lqg_selscan* p) {
  if (!p) return LQG_ERR_NULL;
  if (p->type != LQG_T_F32 && p->type != LQG_T_BF16 && p->type != LQG_T_F16) return LQG_ERR_ARG;
  if (p->B < 1 || p->T < 1 || p->D < 1 || p->D > MAX_STRIDE || p->N < 1 || p->N > 64 || p->G < 1 || p->D % p->G) return LQG_ERR_ARG;
  if (p->chunks < 0 || p->chunks > 64 || (p->channels != 0 && p->channels != 16 && p->channels != 32)) return LQG_ERR_ARG;
  for (const lqg_seq* q : {&p->u, &p->delta, &p->z, &p->Bm, &p->Cm, &p->y})
    if (q->st < 0 || q->st > MAX_STRIDE) return LQG_ERR_ARG;
  for (const lqg_param* q : {&p->A, &p->Dskip, &p->delta_bias})
    if (q->ptr && q->type != LQG_T_F32 && q->type != LQG_T_BF16 && q->type != LQG_T_F16) return LQG_ERR_ARG;
  return 0;
}

// states that the workgroups' shapes have room for (Shape::NP)
long room_of(long N) { return N > 32 ? 64 : N > 16 ? 32 : N > 8 ? 16 : N > 4 ? 8 : 4; }
int tile_of(long N) { return N > 32 ? 8 : 16; }

// How a scan is laid over the card: channels of a workgroup, and pieces that the time axis is cut into.
//
// Time of a pass of w waves over the whole axis, in units of a pass that half fills the 1024 SIMDs: forward two waves of a SIMD overlap, and
// beyond that time grows with their number; backward a SIMD takes one wave at a time (with 9 to 16 states two, so that one alone, which waits
// by itself, leaves time unused).
double pass_time(long N, bool grad, bool narrow, long w) {
  const double q = w / 1024.0;
  if (q <= 0.5) return 1.0;
  if (grad) return q > 1.0 ? std::ceil(q) : N > 8 && N <= 16 ? 1.3 : 1.0;
  if (narrow) return q <= 1.0 ? (N > 4 ? 1.0 : 1.2) : q <= 2.0 ? (N > 4 ? 1.3 : 1.6) : (N > 4 ? 0.6 : 1.0) * q;
  return q <= 1.0 ? 1.1 : q <= 2.0 ? 1.35 : 0.68 * q;
}

// A cut into c pieces adds the pass that leaves the carries of c - 1 of them (0.55 to 0.6 of the main pass's time forward, 0.2 backward), 3 tiles
// a piece before its loads are under way, a launch (8 tiles) and the reading of the carries: the c with the least sum; forward a power of two,
// which leaves whole rounds of workgroups.  Measured, bfloat16 with gate, us at 2048 steps uncut / in 2 / 4 / 8:  forward, 16 channels, N = 16:
// 90 / 82 / 48 / 41 (256 waves uncut), 91 / 103 / 91 / 93 (1024); N = 4: 110 / 100 / 61 / 50 (256), 121 / 126 / 143 / 146 (1024).  Backward
// N = 16: 366 / 258 / 188 / 198 (512), 379 / 325 / 333 / 367 (1024), 516 / 598 / 630 / 700 (2048); N = 24: 572 / 393 / 392 / 439 (512), 592 /
// 689 / 734 / 841 (1024), 1144 / 1026 / 934 / 979 (1100).
struct Cut { double time; long pieces; };
Cut cut(long N, bool grad, bool narrow, long waves, long tiles) {
  Cut best{pass_time(N, grad, narrow, waves), 1};
  const double carry = grad ? 0.2 : narrow ? 0.55 : 0.6;
  for (long c = 2; c <= std::min(64L, tiles / 8); c += grad ? 1 : c) {
    const double main = pass_time(N, grad, narrow, waves * c), before = pass_time(N, grad, narrow, waves * (c - 1));
    const double t = (main + carry * before) * (1.0 / c + 3.0 / tiles) + (8.0 + 0.35 * c) / tiles;
    if (t < best.time) best = {t, c};
  }
  return best;
}

// Forward and up to 32 states a workgroup may have 16 channels instead of 32: twice the waves, each with half the states, in 0.58 to 0.72 of
// the time while they fill the card.  Measured, us with 32 / 16 channels, uncut, 2048 steps x 2048 channels (trials):  N = 4: 179 / 121 (4),
// 192 / 121 (8), 198 / 210 (16), 440 / 386 (32); N = 8: 148 / 119 (4), 190 / 133 (8), 209 / 275 (16); N = 16: 126 / 91 (2), 128 / 126 (4), 177 /
// 204 (8); N = 32: 181 / 119 (2), 186 / 163 (4), 274 / 275 (8).  Over 132 sizes (N = 3 .. 32, 512 to 16384 steps, 32 channels to 32 trials of
// 2048) width and cut chosen so are 2.3 % slower than the best pair in the geometric mean, 24 % at most.
void lay_out(ScanArgs& a, bool grad) {
  const long N = a.p.N, waves = N > 8 ? 4 : N > 4 ? 2 : 1;
  Cut best{};
  auto with = [&](int channels) {
    const long bpg = (a.Dg + channels - 1) / channels;
    const Cut c = cut(N, grad, channels == 16, bpg * a.p.G * a.p.B * waves, a.tiles);
    const double time = c.time * (channels == 32 ? 1.0 : N <= 8 ? 0.68 : N <= 16 ? 0.72 : 0.58);
    if (best.pieces && time >= best.time) return;
    best = {time, c.pieces};
    a.narrow = channels == 16;
    a.bpg = bpg;
  };
  const int asked = grad || N > 32 ? 32 : a.p.channels ? a.p.channels : N <= 4 ? 16 : 0;
  if (asked != 16) with(32);
  if (asked != 32) with(16);
  a.blocks = a.bpg * a.p.G;
  a.chunks = a.p.chunks ? std::min((long)a.p.chunks, a.tiles) : best.pieces;
}

ScanArgs describe(const lqg_selscan* p, bool grad) {
  ScanArgs a{};
  a.p = *p;
  const long TT = tile_of(p->N);
  a.Dg = p->D / p->G;
  a.tiles = (p->T + TT - 1) / TT;
  lay_out(a, grad);
  const long per = (a.tiles + a.chunks - 1) / a.chunks;
  a.chunk = per * TT;
  a.chunks = (a.tiles + per - 1) / per;               // no empty chunk
  return a;
}

long carry_floats(const ScanArgs& a) { return a.chunks > 1 ? a.p.B * a.chunks * (a.p.N + 1) * a.p.D : 0; }

int by_type(int what, const ScanArgs& a, hipStream_t st) {
  if (a.p.type == LQG_T_F32) return ScanOf<float>::run(what, a, st);
  if (a.p.type == LQG_T_BF16) return ScanOf<bf16>::run(what, a, st);
  return ScanOf<f16>::run(what, a, st);
}

bool have(const lqg_selscan* p) { return p->u.ptr && p->delta.ptr && p->A.ptr && p->Bm.ptr && p->Cm.ptr; }

struct GradSpace { long carry, group, rows, cols, mid, total; };
GradSpace grad_space(const ScanArgs& a) {
  GradSpace s;
  s.carry = carry_floats(a);
  s.group = a.blocks * a.p.B * a.p.T * a.p.N;
  s.rows = a.p.B * a.chunks;
  s.cols = (a.p.N + 2) * a.p.D;
  s.mid = row_sum_mid_rows(s.rows, s.cols) * s.cols;
  s.total = s.carry + 2 * s.group + s.rows * s.cols + s.mid;
  return s;
}

}  // namespace

extern "C" size_t lqg_selscan_workspace(const lqg_selscan* p) {
  return check(p) ? 0 : (size_t)carry_floats(describe(p, false)) * sizeof(float);
}
extern "C" size_t lqg_selscan_checkpoint_bytes(const lqg_selscan* p) {
  return check(p) ? 0 : (size_t)(p->B * describe(p, false).tiles * room_of(p->N) * p->D) * sizeof(float);
}
extern "C" size_t lqg_selscan_grad_workspace(const lqg_selscan* p) {
  return check(p) ? 0 : (size_t)grad_space(describe(p, true)).total * sizeof(float);
}

extern "C" int lqg_selective_scan(const lqg_selscan* p, void* workspace, size_t workspace_bytes, void* stream) {
  if (const int rc = check(p)) return rc;
  if (!have(p) || !p->y.ptr) return LQG_ERR_NULL;
  ScanArgs a = describe(p, false);
  const long carry = carry_floats(a);
  if (carry && !workspace) return LQG_ERR_NULL;
  if (workspace_bytes < carry * sizeof(float)) return LQG_ERR_WORKSPACE;
  a.hl = static_cast<float*>(workspace);
  a.sd = a.hl + (carry ? p->B * a.chunks * p->N * p->D : 0);
  return by_type(0, a, (hipStream_t)stream);
}

extern "C" int lqg_selective_scan_grad(const lqg_selscan* p, const lqg_selscan_bars* g, void* workspace, size_t workspace_bytes,
                                       void* stream) {
  if (const int rc = check(p)) return rc;
  if (!g || !have(p) || !p->checkpoints || !workspace) return LQG_ERR_NULL;
  if (g->dy.st < 0 || g->dy.st > MAX_STRIDE) return LQG_ERR_ARG;
  if (!g->dy.ptr || !g->du || !g->ddelta || !g->dBm || !g->dCm || (p->z.ptr && !g->dz)) return LQG_ERR_NULL;
  ScanArgs a = describe(p, true);
  a.g = *g;
  const GradSpace s = grad_space(a);
  if (workspace_bytes < s.total * sizeof(float)) return LQG_ERR_WORKSPACE;
  float* ws = static_cast<float*>(workspace);
  a.hl = ws;
  a.sd = ws + (s.carry ? p->B * a.chunks * p->N * p->D : 0);
  a.partBC = ws + s.carry;
  a.partP = a.partBC + 2 * s.group;
  hipStream_t st = (hipStream_t)stream;
  const long n = p->B * p->T * p->G * 2 * p->N, groups = (n + 255) / 256;
  if (!grid_fits(groups, 256) || !row_sum_fits(s.cols)) return LQG_ERR_ARG;
  if (const int rc = by_type(1, a, st)) return rc;
  const int rc = p->type == LQG_T_F32 ? ScanOf<float>::groups(a, groups, st)
                 : p->type == LQG_T_BF16 ? ScanOf<bf16>::groups(a, groups, st) : ScanOf<f16>::groups(a, groups, st);
  if (rc) return rc;
  RowSum r{a.partP, s.rows, s.cols, a.partP + s.rows * s.cols};
  RowSumOut o{};
  o.ptr[0] = g->dA, o.type[0] = p->A.type, o.major[0] = p->N, o.minor[0] = p->D;
  o.ptr[1] = g->dD, o.type[1] = p->Dskip.type, o.major[1] = 1, o.minor[1] = p->D;
  o.ptr[2] = g->ddelta_bias, o.type[2] = p->delta_bias.type, o.major[2] = 1, o.minor[2] = p->D;
  o.begin[1] = p->N * p->D, o.begin[2] = (p->N + 1) * p->D, o.begin[3] = s.cols;
  return (int)row_sum(r, o, st);
}

extern "C" int lqg_selective_scan_step(const lqg_selscan* p, float* state, void* stream) {
  if (const int rc = check(p)) return rc;
  if (p->T != 1) return LQG_ERR_ARG;
  if (!have(p) || !p->y.ptr || !state) return LQG_ERR_NULL;
  ScanArgs a = describe(p, false);
  hipStream_t st = (hipStream_t)stream;
  if (p->type == LQG_T_F32) return ScanOf<float>::step(a, state, st);
  if (p->type == LQG_T_BF16) return ScanOf<bf16>::step(a, state, st);
  return ScanOf<f16>::step(a, state, st);
}
#endif
