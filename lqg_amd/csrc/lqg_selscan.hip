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
  if (p->chunks < 0 || p->chunks > 64) return LQG_ERR_ARG;
  for (const lqg_seq* q : {&p->u, &p->delta, &p->z, &p->Bm, &p->Cm, &p->y})
    if (q->st < 0 || q->st > MAX_STRIDE) return LQG_ERR_ARG;
  for (const lqg_param* q : {&p->A, &p->Dskip, &p->delta_bias})
    if (q->ptr && q->type != LQG_T_F32 && q->type != LQG_T_BF16 && q->type != LQG_T_F16) return LQG_ERR_ARG;
  return 0;
}

// states that the workgroups' shapes have room for (Shape::NP)
long room_of(long N) { return N > 32 ? 64 : N > 16 ? 32 : N > 8 ? 16 : N > 4 ? 8 : 4; }
int tile_of(long N) { return N > 32 ? 8 : 16; }

// Time of a pass of w waves over the whole axis, in units of one that half fills the 1024 SIMDs: as many rounds as fill them, and a tenth
// more when every SIMD is taken.  Forward with 5 to 8 states workgroups of two waves share SIMDs early, and backward with 9 to 16 states
// registers let two waves share one, so that one alone, which waits by itself, leaves time unused (in both 1.3).
double pass_time(long N, bool grad, long w) {
  const double q = w / 1024.0;
  const bool shared = grad ? N > 8 && N <= 16 : N > 4 && N <= 8;
  if (q <= 0.5) return 1.0;
  if (q <= 1.0) return shared ? 1.3 : 1.1;
  if (shared && !grad) return q <= 2.0 ? 1.6 : 0.96 * q;
  return std::ceil(q);
}

// Pieces of the time axis.  A cut into c adds the pass that leaves the carries of c - 1 of them (0.55 of the main pass's time forward, 0.2
// backward), 3 tiles a piece before its loads are under way, and a launch (6 tiles): the c with the least sum.  Measured, bfloat16 with
// gate, us uncut / in 2 / 4 / 8 at 2048 steps:  forward N = 16: 126 / 115 / 88 / 88 (512 waves uncut), 128 / 138 / 135 / 143 (1024);
// N = 8: 149 / 151 / 98 / 107 (512), 192 / 179 / 170 / 198 (1024).  Backward N = 16: 366 / 258 / 188 / 198 (512), 379 / 325 / 333 / 367
// (1024), 516 / 598 / 630 / 700 (2048); N = 24: 572 / 393 / 392 / 439 (512), 592 / 689 / 734 / 841 (1024), 1144 / 1026 / 934 / 979 (1100).
// Over 164 such rows (N = 4 .. 64, 512 to 6000 steps, 64 to 2048 waves) the choice is 1.3 % slower than the best cut (geometric mean, 25 %
// at most); filling the SIMDs up to a threshold of waves was 6.8 % (54 %).
long pieces(long N, bool grad, long waves, long tiles) {
  long best = 1;
  double least = pass_time(N, grad, waves);
  for (long c = 2; c <= std::min(64L, tiles / 8); ++c) {
    const double t = (pass_time(N, grad, waves * c) + (grad ? 0.2 : 0.55) * pass_time(N, grad, waves * (c - 1))) * (1.0 / c + 3.0 / tiles) +
                     6.0 / tiles;
    if (t < least) least = t, best = c;
  }
  return best;
}

ScanArgs describe(const lqg_selscan* p, bool grad) {
  ScanArgs a{};
  a.p = *p;
  const long TT = tile_of(p->N);
  a.Dg = p->D / p->G;
  a.bpg = (a.Dg + CHANNELS - 1) / CHANNELS;
  a.blocks = a.bpg * p->G;
  a.tiles = (p->T + TT - 1) / TT;
  const long waves = a.blocks * p->B * (p->N > 8 ? 4 : p->N > 4 ? 2 : 1);
  a.chunks = p->chunks ? std::min((long)p->chunks, a.tiles) : pieces(p->N, grad, waves, a.tiles);
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
