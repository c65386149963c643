// Linear block: y = act(x W^T + bias) + residual over rows of channels (a pointwise convolution over
// channels-last voxels), and its gradient.
//
//   z = x W^T + b            y = act(z) + r
//   dz = dy * act'(z)        dx = dz W        dW = dz^T x        db = sum over rows of dz        dr = dy
//
// The epilogue runs on the accumulators, so z, act(z) and the sum with r never pass through memory,
// apart from z itself where a backward pass will want it.
#include <climits>

#include "mat.h"

namespace cg {
namespace {

constexpr int kTile = 64;

int dt_bytes(int dt) { return dt == CGAN3D_DT_F32 ? 4 : 2; }

// Splits of the summed axis: as many as fill the card twice, each at least 256 values long.
int mat_splits(long long I, long long J, long long K) {
  const long long tiles = std::max(1LL, ((I + kTile - 1) / kTile) * ((J + kTile - 1) / kTile));
  const long long want = 2LL * cu_count() / tiles, most = K / 256;
  return (int)std::max(1LL, std::min({want, most, 1024LL}));
}
long long mat_ws_bytes(long long I, long long J, long long K) {
  const int s = mat_splits(I, J, K);
  return s > 1 ? (long long)s * I * J * 4 : 0;
}

template <typename T, bool AT, bool BT>
void mat_run_t(MatArgs p, void* ws, hipStream_t st) {
  if (p.I == 0 || p.J == 0) return;
  int splits = mat_splits(p.I, p.J, p.K);
  const long long steps = (p.K + 31) / 32;
  p.kchunk = std::max(1LL, (steps + splits - 1) / splits) * 32;
  splits = (int)std::max(1LL, (p.K + p.kchunk - 1) / p.kchunk);
  p.part = splits > 1 ? static_cast<float*>(ws) : nullptr;
  const long long ti = (p.I + kTile - 1) / kTile;
  p.tj = (p.J + kTile - 1) / kTile;
  launch(mat_kernel<T, AT, BT, kTile, kTile>, dim3((unsigned)(ti * p.tj), splits), dim3(256), 0, st, p);
  if (splits > 1) {
    const long long blocks = std::min((p.I * p.J + 255) / 256, 8192LL);
    launch(mat_join_kernel<T>, dim3((unsigned)blocks), dim3(256), 0, st, p, splits);
  }
}
template <bool AT, bool BT>
void mat_run(int dt, const MatArgs& p, void* ws, hipStream_t st) {
  if (dt == CGAN3D_DT_F32) mat_run_t<float, AT, BT>(p, ws, st);
  else if (dt == CGAN3D_DT_BF16) mat_run_t<bf16_t, AT, BT>(p, ws, st);
  else mat_run_t<f16_t, AT, BT>(p, ws, st);
}

// dz = dy * act'(z) and the column sums of dz (in 32 bits, before its rounding): 64 columns x 4 rows a
// block, `rows` rows of them; part [blockIdx.y][n].
template <typename T>
__global__ __launch_bounds__(256) void act_grad_kernel(const T* __restrict__ dy, long long lddy,
                                                       const typename PreT<T>::type* __restrict__ pre, T* __restrict__ dz,
                                                       float* __restrict__ part, long long rows, int n, long long chunk,
                                                       int act, float slope) {
  __shared__ float red[4][64];
  const int c = threadIdx.x & 63, r = threadIdx.x >> 6;
  const long long j = (long long)blockIdx.x * 64 + c;
  const long long i1 = std::min(rows, ((long long)blockIdx.y + 1) * chunk);
  float s = 0.f;
  if (j < n) {
    for (long long i = (long long)blockIdx.y * chunk + r; i < i1; i += 4) {
      float v = to_f(dy[i * lddy + j]);
      if (act != CGAN3D_ACT_NONE) {
        v *= mat_act_grad(to_f(pre[i * n + j]), act, slope);
        dz[i * n + j] = from_f<T>(v);
      }
      s += v;
    }
  }
  red[r][c] = s;
  __syncthreads();
  if (r == 0 && j < n && part) part[(long long)blockIdx.y * n + j] = (red[0][c] + red[1][c]) + (red[2][c] + red[3][c]);
}

template <typename T>
__global__ __launch_bounds__(256) void bias_join_kernel(const float* __restrict__ part, int nb, int n, T* __restrict__ db) {
  const long long j = (long long)blockIdx.x * 256 + threadIdx.x;
  if (j >= n) return;
  double s = 0.;
  for (int b = 0; b < nb; ++b) s += part[(long long)b * n + j];
  db[j] = from_f<T>((float)s);
}

long long act_chunk(long long rows, int n) {
  const long long cols = (n + 63) / 64;
  const long long want = std::max(1LL, 8LL * cu_count() / cols);
  return std::max(16LL, (rows + want - 1) / want);
}

template <typename T>
void act_grad_run(const cgan3d_linear_args* a, T* dz, float* part, hipStream_t st) {
  const long long chunk = act_chunk(a->rows, a->n), nb = (a->rows + chunk - 1) / chunk;
  if (nb > 0 && a->n > 0)
    launch(act_grad_kernel<T>, dim3((a->n + 63) / 64, (unsigned)nb), dim3(256), 0, st, static_cast<const T*>(a->dy),
           (long long)a->lddy, static_cast<const typename PreT<T>::type*>(a->preact), dz, part, (long long)a->rows,
           a->n, chunk, a->act, a->slope);
  if (a->dbias && a->n > 0)
    launch(bias_join_kernel<T>, dim3((a->n + 255) / 256), dim3(256), 0, st, (const float*)part, (int)nb, a->n,
           static_cast<T*>(a->dbias));
}

long long up256(long long v) { return (v + 255) / 256 * 256; }

struct Bwd {  // workspace layout of the backward pass
  long long dz, part, mat, total;
};
Bwd bwd_layout(const cgan3d_linear_args* a) {
  Bwd w;
  w.dz = 0;
  long long at = a->act != CGAN3D_ACT_NONE ? up256(a->rows * a->n * dt_bytes(a->dtype)) : 0;
  w.part = at;
  const long long chunk = act_chunk(a->rows, a->n);
  if (a->dbias) at += up256((a->rows + chunk - 1) / chunk * a->n * 4);
  w.mat = at;
  const long long m1 = a->dx ? mat_ws_bytes(a->rows, a->k, a->n) : 0, m2 = a->dw ? mat_ws_bytes(a->n, a->k, a->rows) : 0;
  w.total = at + std::max(m1, m2);  // the two products run one after the other
  return w;
}

const char* lin_check(const cgan3d_linear_args* a, bool bwd) {
  if (!a) return "null args";
  if (a->dtype < CGAN3D_DT_F32 || a->dtype > CGAN3D_DT_F16) return "unknown dtype";
  if (a->rows < 0 || a->k < 0 || a->n < 0) return "negative size";
  if (a->rows > (1LL << 40)) return "too many rows";
  const long long t = (a->rows + kTile - 1) / kTile, u = ((long long)std::max(a->k, a->n) + kTile - 1) / kTile;
  if (t * u > INT_MAX || u * u > INT_MAX) return "too many tiles for one launch";
  if (a->act < CGAN3D_ACT_NONE || a->act > CGAN3D_ACT_SILU || a->act == CGAN3D_ACT_NEG_DTANH)
    return "activation must be none, relu, lrelu, tanh, gelu or silu";
  if ((a->k > 0 && a->rows > 0 && !a->x) || (a->k > 0 && a->n > 0 && !a->w)) return "null operand";
  if (a->ldx < a->k || a->ldw < a->k) return "row stride smaller than the row";
  const bool out = a->rows > 0 && a->n > 0;
  if (!bwd) {
    if (out && !a->y) return "null output";
    if (a->ldy < a->n || (a->residual && a->ldr < a->n)) return "row stride smaller than the row";
  } else {
    if (out && !a->dy) return "null dy";
    if (a->lddy < a->n || (a->dx && a->lddx < a->k)) return "row stride smaller than the row";
    if (out && a->act != CGAN3D_ACT_NONE && !a->preact) return "the activation's gradient needs preact";
  }
  return nullptr;
}

struct Span {
  uintptr_t lo, hi;
};
Span span(const void* p, long long rows, long long cols, long long ld, int e) {
  const uintptr_t b = reinterpret_cast<uintptr_t>(p);
  if (!p || rows <= 0 || cols <= 0) return {0, 0};
  return {b, b + ((rows - 1) * ld + cols) * e};
}
bool meet(Span a, Span b) { return a.lo < b.hi && b.lo < a.hi; }

}  // namespace

long long mat_f32_ws_bytes(long long I, long long J, long long K) { return mat_ws_bytes(I, J, K); }
void mat_f32(bool at, bool bt, const MatArgs& p, void* ws, hipStream_t st) {
  if (at) mat_run_t<float, true, true>(p, ws, st);
  else if (bt) mat_run_t<float, false, true>(p, ws, st);
  else mat_run_t<float, false, false>(p, ws, st);
}

}  // namespace cg

using namespace cg;

extern "C" int64_t cgan3d_linear_fwd_ws_bytes(const cgan3d_linear_args* a) {
  if (const char* e = lin_check(a, false)) {
    set_error("cgan3d_linear_fwd_ws_bytes: %s", e);
    return -1;
  }
  return mat_ws_bytes(a->rows, a->n, a->k);
}

extern "C" int cgan3d_linear_fwd(const cgan3d_linear_args* a, void* ws, int64_t ws_bytes, void* stream) try {
  const char* e = lin_check(a, false);
  CG_CHECK_ARG(!e, "cgan3d_linear_fwd: %s", e);
  const long long need = mat_ws_bytes(a->rows, a->n, a->k);
  CG_CHECK_ARG(ws_bytes >= need && (need == 0 || (ws && reinterpret_cast<uintptr_t>(ws) % 16 == 0)),
               "cgan3d_linear_fwd: workspace of %lld bytes (16-byte aligned) needed, got %lld", need, (long long)ws_bytes);
  const int b = dt_bytes(a->dtype), pb = a->dtype == CGAN3D_DT_F32 ? 4 : 2;
  const Span y = span(a->y, a->rows, a->n, a->ldy, b), z = span(a->preact, a->rows, a->n, a->n, pb);
  const Span x = span(a->x, a->rows, a->k, a->ldx, b), w = span(a->w, a->n, a->k, a->ldw, b);
  const Span r = span(a->residual, a->rows, a->n, a->ldr, b), bi = span(a->bias, 1, a->n, a->n, b);
  CG_CHECK_ARG(!meet(y, x) && !meet(y, w) && !meet(y, bi) && !meet(y, z) && !meet(z, x) && !meet(z, w) && !meet(z, r) &&
                   !meet(z, bi) && (!meet(y, r) || (a->y == a->residual && a->ldy == a->ldr)),
               "cgan3d_linear_fwd: an output overlaps an operand (y may be the residual itself)");
  MatArgs p = {};
  p.a = a->x; p.lda = a->ldx;
  p.b = a->w; p.ldb = a->ldw;
  p.I = a->rows; p.J = a->n; p.K = a->k;
  p.e = {a->bias, a->residual, a->ldr, a->preact, a->y, a->ldy, 1.f, 1.f, a->act, a->slope};
  mat_run<false, false>(a->dtype, p, ws, (hipStream_t)stream);
  CG_LAUNCH_CHECK("cgan3d_linear_fwd");
  return CGAN3D_OK;
} catch (...) {
  set_error("cgan3d_linear_fwd: out of host memory");
  return CGAN3D_EHIP;
}

extern "C" int64_t cgan3d_linear_bwd_ws_bytes(const cgan3d_linear_args* a) {
  if (const char* e = lin_check(a, true)) {
    set_error("cgan3d_linear_bwd_ws_bytes: %s", e);
    return -1;
  }
  return bwd_layout(a).total;
}

extern "C" int cgan3d_linear_bwd(const cgan3d_linear_args* a, void* ws, int64_t ws_bytes, void* stream) try {
  const char* e = lin_check(a, true);
  CG_CHECK_ARG(!e, "cgan3d_linear_bwd: %s", e);
  const Bwd l = bwd_layout(a);
  CG_CHECK_ARG(ws_bytes >= l.total && (l.total == 0 || (ws && reinterpret_cast<uintptr_t>(ws) % 16 == 0)),
               "cgan3d_linear_bwd: workspace of %lld bytes (16-byte aligned) needed, got %lld", l.total,
               (long long)ws_bytes);
  const int b = dt_bytes(a->dtype);
  const Span in[] = {span(a->x, a->rows, a->k, a->ldx, b), span(a->w, a->n, a->k, a->ldw, b),
                     span(a->dy, a->rows, a->n, a->lddy, b),
                     a->act != CGAN3D_ACT_NONE ? span(a->preact, a->rows, a->n, a->n, b) : Span{0, 0}};
  const Span out[] = {span(a->dx, a->rows, a->k, a->lddx, b), span(a->dw, a->n, a->k, a->k, b),
                      span(a->dbias, 1, a->n, a->n, b)};
  for (int o = 0; o < 3; ++o) {
    for (const Span& s : in) CG_CHECK_ARG(!meet(out[o], s), "cgan3d_linear_bwd: a gradient overlaps an operand");
    for (int q = 0; q < o; ++q) CG_CHECK_ARG(!meet(out[o], out[q]), "cgan3d_linear_bwd: two gradients overlap");
  }
  hipStream_t st = (hipStream_t)stream;
  char* base = static_cast<char*>(ws);
  const bool act = a->act != CGAN3D_ACT_NONE;
  void* dz = act ? base + l.dz : nullptr;
  float* part = a->dbias ? reinterpret_cast<float*>(base + l.part) : nullptr;
  if (a->dbias || (act && (a->dx || a->dw))) {
    if (a->dtype == CGAN3D_DT_F32) act_grad_run<float>(a, (float*)dz, part, st);
    else if (a->dtype == CGAN3D_DT_BF16) act_grad_run<bf16_t>(a, (bf16_t*)dz, part, st);
    else act_grad_run<f16_t>(a, (f16_t*)dz, part, st);
  }
  MatArgs p = {};
  p.a = act ? dz : a->dy;
  p.lda = act ? a->n : a->lddy;
  p.e.alpha = 1.f;
  if (a->dx) {
    MatArgs q = p;
    q.b = a->w; q.ldb = a->ldw;
    q.I = a->rows; q.J = a->k; q.K = a->n;
    q.e.out = a->dx; q.e.ldo = a->lddx;
    mat_run<false, true>(a->dtype, q, base + l.mat, st);
  }
  if (a->dw) {
    MatArgs q = p;
    q.b = a->x; q.ldb = a->ldx;
    q.I = a->n; q.J = a->k; q.K = a->rows;
    q.e.out = a->dw; q.e.ldo = a->k;
    mat_run<true, true>(a->dtype, q, base + l.mat, st);
  }
  CG_LAUNCH_CHECK("cgan3d_linear_bwd");
  return CGAN3D_OK;
} catch (...) {
  set_error("cgan3d_linear_bwd: out of host memory");
  return CGAN3D_EHIP;
}
