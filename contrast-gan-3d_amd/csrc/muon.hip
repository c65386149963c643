// Orthogonalised updates: the Newton-Schulz iteration on a list of matrices, and the Muon optimiser's
// step over a parameter arena.
//
//   X_0 = G / (|G|_F + eps)        (over the short side: a tall G is taken transposed)
//   A = X X^T,  B = b A + c A A,  X <- a X + B X        `steps` times
//
// which applies the odd quintic a s + b s^3 + c s^5 to every singular value s and leaves the singular
// vectors alone; with (3.4445, -4.7750, 2.0315) five steps bring all but the smallest close to 1.
//
// Muon (arena segments that are matrices):  m <- m + (1 - mu)(g - m),  u = g + mu (m - g) (Nesterov) or m,
//   p <- p (1 - lr wd) - lr scale NS(u);   segments that are vectors: Adam with their own rate.
//
// The norm is summed in 64 bits (a gradient of 1e-25 squares to nothing in 32).  The iteration keeps f32's
// accuracy on two f16 planes per matrix (planes.h): the iterates are bounded (|X| <= 1.2, |A| <= 1.5 with the
// coefficients above), so a fixed power of two keeps hi + lo within f16's range: X at 2^12 (an entry of a
// large orthogonal matrix, ~2^-6, and one of a fresh gradient's, ~2^-12, both keep 22 bits), A and B at 2^10.
// A matrix far below eps starts at |X| = |G| / eps << 1 and grows by at most a factor per step that planes_hold finds
// (a = 3.4445 here): its planes are held at a further 2^e, e from the norm and smaller by that factor's exponent with
// every step, which the epilogues take back (A and B are needed to 2^-34 beside a alone, so theirs need none).
// The first term a X is added in the epilogue from X's own planes: as part of B it would lose the
// products of the low planes, which directions that start near zero then carry a^5 = 485 times larger.
// Coefficients that let the iterates leave that range, and no steps at all, take the f32 products of mat.h.
// A and B are symmetric: the lower triangle's tiles are computed and stored twice.
#include <climits>
#include <cmath>

#include "planes.h"

namespace cg {
namespace {

long long up256(long long v) { return (v + 255) / 256 * 256; }

constexpr int kNormBlocks = 256;  // partial sums per matrix
constexpr int kList = 24;        // segments a launch takes by value

// hyper (device): see include/cgan3d.h cgan3d_muon_step
enum { H_LR, H_MU, H_WD, H_NESTEROV, H_STEP, H_CLIP, H_VLR, H_VB1, H_VB2, H_VEPS, H_COUNT };

struct Mat {
  const void* g;
  void* out;  // orthogonalize: the result; muon: the parameter
  long long ldg, ldo;
  int rows, cols;
  float scale;  // muon: factor of lr
  float* x;     // iterate, [short][long]
  double* part;
};

static_assert(kNormBlocks == 256, "the partial sums are added by a block of 256 threads");
__device__ __forceinline__ double block_sum_d(double v) {
  __shared__ double red[4];
  v = wave_sum_d(v);
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
  __syncthreads();
  return (red[0] + red[1]) + (red[2] + red[3]);
}

struct MatList {
  Mat m[kList];
};
struct SegList {
  cgan3d_muon_seg s[kList];
  long long u[kList];  // offset of the segment's update in the workspace
  int mat[kList];      // index of the matrix (its partial sums), -1: a vector
};

// sum of squares of a matrix, kNormBlocks partial sums; 16 bytes a lane where its rows follow each other
template <typename T>
__global__ __launch_bounds__(256) void norm_kernel(MatList l) {
  constexpr int V = MatT<T>::VEC;
  typedef T vecT __attribute__((ext_vector_type(V)));
  const Mat& m = l.m[blockIdx.y];
  const T* g = static_cast<const T*>(m.g);
  const long long total = (long long)m.rows * m.cols, tid = (long long)blockIdx.x * 256 + threadIdx.x;
  double s = 0.;
  if (m.ldg == m.cols || m.rows == 1) {
    for (long long q = tid; q < total / V; q += kNormBlocks * 256LL) {
      const vecT x = load_v<vecT>(g + q * V);
#pragma unroll
      for (int e = 0; e < V; ++e) {
        const double v = to_f(x[e]);
        s += v * v;
      }
    }
    if (tid < total % V) {
      const double v = to_f(g[total / V * V + tid]);
      s += v * v;
    }
  } else {
    for (long long q = tid; q < total; q += kNormBlocks * 256LL) {
      const long long i = q / m.cols;
      const double v = to_f(g[i * m.ldg + (q - i * m.cols)]);
      s += v * v;
    }
  }
  s = block_sum_d(s);
  if (threadIdx.x == 0) m.part[blockIdx.x] = s;
}

// momentum and the update's squares (matrices), Adam (vectors)
__global__ __launch_bounds__(256) void muon_moment_kernel(SegList l, float* __restrict__ param,
                                                          const float* __restrict__ grad, float* __restrict__ mom,
                                                          float* __restrict__ sq, const float* __restrict__ hyper,
                                                          float* __restrict__ u, double* __restrict__ part) {
  const cgan3d_muon_seg sg = l.s[blockIdx.y];
  const long long total = sg.rows > 0 ? sg.rows * sg.cols : sg.cols, base = sg.offset;
  if (sg.rows == 0) {
    const float h[6] = {hyper[H_VLR], hyper[H_VB1], hyper[H_VB2], hyper[H_VEPS], 0.f, hyper[H_CLIP]};
    const AdamK k = adam_k(h, hyper[H_STEP] + 1.f);
    for (long long q = (long long)blockIdx.x * 256 + threadIdx.x; q < total; q += kNormBlocks * 256LL)
      adam_elem(k, param, grad, mom, sq, base + q);
    return;
  }
  const float mu = hyper[H_MU];
  const bool nest = hyper[H_NESTEROV] != 0.f;
  double s = 0.;
  for (long long q = (long long)blockIdx.x * 256 + threadIdx.x; q < total; q += kNormBlocks * 256LL) {
    const float g = grad[base + q];
    float m = mom[base + q];
    m += (1.f - mu) * (g - m);
    mom[base + q] = m;
    const float v = nest ? g + mu * (m - g) : m;
    u[l.u[blockIdx.y] + q] = v;
    s += (double)v * v;
  }
  s = block_sum_d(s);
  if (threadIdx.x == 0) part[(long long)l.mat[blockIdx.y] * kNormBlocks + blockIdx.x] = s;
}

// The exponent e of the planes' further factor: x = |G| / (|G| + eps) in [1/2, 1) as they hold it, 0 where it is larger
// or no number
__device__ __forceinline__ int start_exponent(double x) {
  return x > 0. && x < 0.5 ? -ilogb(x) - 1 : 0;
}

template <typename T>
__global__ __launch_bounds__(256) void scale_kernel(MatList l, float eps) {
  const Mat& m = l.m[blockIdx.y];
  const double s = block_sum_d(m.part[threadIdx.x]);  // one partial sum a thread
  const double inv = 1. / (sqrt(s) + (double)eps);  // the norm of finite values may be beyond f32
  const T* g = static_cast<const T*>(m.g);
  const bool tall = m.rows > m.cols;
  const int lng = tall ? m.rows : m.cols;
  const long long total = (long long)m.rows * m.cols;
  for (long long q = (long long)blockIdx.x * 256 + threadIdx.x; q < total; q += gridDim.x * 256LL) {
    const long long i = q / lng, t = q - i * lng;
    m.x[q] = (float)(to_f(tall ? g[t * m.ldg + i] : g[i * m.ldg + t]) * inv);
  }
}

template <typename T>
__global__ __launch_bounds__(256) void ortho_out_kernel(MatList l) {
  const Mat& m = l.m[blockIdx.y];
  const bool tall = m.rows > m.cols;
  const long long total = (long long)m.rows * m.cols;
  T* o = static_cast<T*>(m.out);
  for (long long q = (long long)blockIdx.x * 256 + threadIdx.x; q < total; q += gridDim.x * 256LL) {
    const long long i = q / m.cols, j = q - i * m.cols;
    o[i * m.ldo + j] = from_f<T>(tall ? m.x[j * m.rows + i] : m.x[q]);
  }
}

__global__ __launch_bounds__(256) void muon_apply_kernel(MatList l, const float* __restrict__ hyper) {
  const Mat& m = l.m[blockIdx.y];
  const bool tall = m.rows > m.cols;
  const long long total = (long long)m.rows * m.cols;
  float* p = static_cast<float*>(m.out);
  const float lr = hyper[H_LR], keep = 1.f - lr * hyper[H_WD], rate = lr * m.scale, clip = hyper[H_CLIP];
  for (long long q = (long long)blockIdx.x * 256 + threadIdx.x; q < total; q += gridDim.x * 256LL) {
    const long long i = q / m.cols, j = q - i * m.cols;
    float v = p[q] * keep - rate * (tall ? m.x[j * m.rows + i] : m.x[q]);
    if (clip > 0.f) v = fminf(fmaxf(v, -clip), clip);
    p[q] = v;
  }
}

// --- the iteration on planes ---
constexpr int kJobs = 12;  // matrices in flight
constexpr float kXs = 4096.f, kAs = 1024.f;

// A = X X^T (beta 0) or B = b A + c A A, from sums in the operands' scales to planes in A's
struct GramEpi {
  static constexpr bool STAGED = false;
  f16_t* out;
  const f16_t* in;  // A's planes
  int ld, n;        // row stride, side
  long long plane;  // elements between planes
  float alpha, beta;
  const int* expo;  // A: X's start exponent (B: null)
  int drop;         // by how much it has fallen
  __device__ __forceinline__ int begin() const { return expo ? *expo : 0; }
  // called by whole waves: lane l has row l % 16 and columns 4 (l / 16) .. + 3 of a 16 x 16 block
  __device__ __forceinline__ void put(int i, int j, f32x4_m v, int jn, bool mirror, int start) const {
    const long long o = (long long)i * ld + j;
    const float alpha = ldexpf(this->alpha, -2 * max(start - drop, 0));
    const int lane = threadIdx.x & 63, t = lane & 3;
    if (jn >= 4) {
      f16x4_m h, l;
      f32x4_m x = alpha * v;
      if (in) {
        const f16x4_m a = *reinterpret_cast<const f16x4_m*>(in + o), c = *reinterpret_cast<const f16x4_m*>(in + plane + o);
#pragma unroll
        for (int r = 0; r < 4; ++r) x[r] += beta * ((float)a[r] + (float)c[r]);
      }
      unsigned w[4];
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        f16_t s[2];
        split2(x[r], s);
        h[r] = s[0];
        l[r] = s[1];
        w[r] = __builtin_bit_cast(unsigned short, s[0]) | (unsigned)__builtin_bit_cast(unsigned short, s[1]) << 16;
      }
      *reinterpret_cast<f16x4_m*>(out + o) = h;
      *reinterpret_cast<f16x4_m*>(out + plane + o) = l;
      if (!mirror) return;
      if ((i & ~15) + 16 <= n) {
        // 4 x 4 transposes in the quads of lanes (rows i .. i + 3 of four columns): lane t ends up with column
        // j + t of the quad's four rows, which are neighbours in the mirrored row
#define CG_SWAP(A, B, CTRL, BIT)                                                                              \
  {                                                                                                           \
    const unsigned pa = __builtin_amdgcn_mov_dpp(A, CTRL, 0xf, 0xf, true),                                    \
                   pb = __builtin_amdgcn_mov_dpp(B, CTRL, 0xf, 0xf, true);                                    \
    A = (t & BIT) ? pb : A;                                                                                   \
    B = (t & BIT) ? B : pa;                                                                                   \
  }
        CG_SWAP(w[0], w[1], 0xB1, 1)
        CG_SWAP(w[2], w[3], 0xB1, 1)
        CG_SWAP(w[0], w[2], 0x4E, 2)
        CG_SWAP(w[1], w[3], 0x4E, 2)
#undef CG_SWAP
        const long long m = (long long)(j + t) * ld + (i & ~3);
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          h[r] = __builtin_bit_cast(f16_t, (unsigned short)w[r]);
          l[r] = __builtin_bit_cast(f16_t, (unsigned short)(w[r] >> 16));
        }
        *reinterpret_cast<f16x4_m*>(out + m) = h;
        *reinterpret_cast<f16x4_m*>(out + plane + m) = l;
      } else {
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const long long m = (long long)(j + r) * ld + i;
          out[m] = h[r];
          out[plane + m] = l[r];
        }
      }
      return;
    }
    // the last columns of the last tile, which is on the diagonal: no mirror
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      if (r >= jn) break;
      float x = alpha * v[r];
      if (in) x += beta * ((float)in[o + r] + (float)in[plane + o + r]);
      f16_t s[2];
      split2(x, s);
      out[o + r] = s[0];
      out[plane + o + r] = s[1];
    }
  }
};

// X <- a X + B X: to planes, or where it is the last step to the result / the parameter
struct StepEpi {
  static constexpr bool STAGED = true;
  f16_t* out;
  const f16_t* in;  // X's planes
  long long plane;
  int ld;
  int mode;  // 0 planes, 1 + dtype: the result, 4: the parameter
  float alpha, beta;
  void* res;
  long long ldr;
  int tall;
  float scale;
  const float* hyper;
  const int* expo;  // X's start exponent
  int drop, next;   // by how much it has fallen, and will have in the result

  __device__ __forceinline__ int begin() const { return *expo; }
  __device__ __forceinline__ bool turned() const { return tall && mode; }

  // the last step's values x at offset d of the result or the parameter, n of them
  __device__ __forceinline__ void finish(long long d, f32x4_m x, int n) const {
    x *= 1.f / kXs;
    if (mode == 1 + CGAN3D_DT_F32) {
      store4(static_cast<float*>(res) + d, x, n);
    } else if (mode == 1 + CGAN3D_DT_BF16) {
      store4(static_cast<bf16_t*>(res) + d, x, n);
    } else if (mode == 1 + CGAN3D_DT_F16) {
      store4(static_cast<f16_t*>(res) + d, x, n);
    } else {
      float* p = static_cast<float*>(res) + d;
      const float lr = hyper[H_LR], clip = hyper[H_CLIP], keep = 1.f - lr * hyper[H_WD], rate = lr * scale;
      f32x4_m w;
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        w[r] = r < n ? p[r] * keep - rate * x[r] : 0.f;
        if (clip > 0.f) w[r] = fminf(fmaxf(w[r], -clip), clip);
      }
      store4(p, w, n);
    }
  }
  // four columns from j of rows i, i + STEP, .. + 3 STEP: every load before the first store
  template <int STEP> __device__ __forceinline__ void put4(int i, int j, f32x4_m* v, int I, int jn, int start) const {
    const int ex = max(start - next, 0) - max(start - drop, 0);
    f16x4_m a[4], c[4];
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const long long o = (long long)min(i + u * STEP, I - 1) * ld + j;  // rows of whole 32s: four columns are there
      a[u] = *reinterpret_cast<const f16x4_m*>(in + o);
      c[u] = *reinterpret_cast<const f16x4_m*>(in + plane + o);
    }
#pragma unroll
    for (int u = 0; u < 4; ++u) {
#pragma unroll
      for (int r = 0; r < 4; ++r) v[u][r] = ldexpf(alpha * v[u][r] + beta * ((float)a[u][r] + (float)c[u][r]), ex);
      if (i + u * STEP >= I || turned()) continue;
      if (mode == 0) {
        f16x4_m h, l;
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          f16_t s[2];
          split2(r < jn ? v[u][r] : 0.f, s);  // the padding stays zero
          h[r] = s[0];
          l[r] = s[1];
        }
        const long long o = (long long)(i + u * STEP) * ld + j;
        *reinterpret_cast<f16x4_m*>(out + o) = h;
        *reinterpret_cast<f16x4_m*>(out + plane + o) = l;
      } else {
        finish((i + u * STEP) * ldr + j, v[u], jn);
      }
    }
  }
  // column j of the result, rows i .. i + 3 of the iterate
  __device__ __forceinline__ void put_turned(int i, int j, f32x4_m v, int in_) const { finish(j * ldr + i, v, in_); }
  __device__ __forceinline__ void put(int i, int j, f32x4_m v, int jn, bool, int start) const {
    f32x4_m w[4] = {v};
    put4<1>(i, j, w, i + 1, jn, start);
    if (turned())
#pragma unroll
      for (int r = 0; r < 4; ++r)
        if (r < jn) finish((j + r) * ldr + i, f32x4_m{w[0][r], 0.f, 0.f, 0.f}, 1);
  }
};

struct PlaneMat {  // one matrix's planes in the workspace
  f16_t *x, *y, *a, *b;
  int* expo;  // start exponent
  int s, l, lda, ldx;  // short and long side, row strides of A / B and X / Y (multiples of 32)
};
struct PlaneMats {
  PlaneMat p[kJobs];
};

// X's planes from G, 32 x 64 of them at a time (a tall G is turned in LDS); the padding of the rows is zeroed
// in all four, once: the products read it, nothing else is written there
template <typename T>
__global__ __launch_bounds__(256) void planes_kernel(MatList l, PlaneMats pm, float eps) {
  __shared__ float tile[64][33];
  const Mat& m = l.m[blockIdx.y];
  const PlaneMat& p = pm.p[blockIdx.y];
  const double s = block_sum_d(m.part[threadIdx.x]);  // one partial sum a thread
  const double size = sqrt(s), inv = 1. / (size + (double)eps);
  const int e = start_exponent(size * inv);
  // from G to the planes, the rest of a power of two apart: either may be beyond f32 where G is
  int to;
  const float rest = (float)frexp(kXs * inv, &to);
  to += e;
  if (blockIdx.x == 0 && threadIdx.x == 0) *p.expo = e;
  const T* g = static_cast<const T*>(m.g);
  const bool tall = m.rows > m.cols;
  const long long xp = (long long)p.s * p.ldx, ap = (long long)p.s * p.lda;
  const int nc = (p.ldx + 63) / 64, nt = (p.s + 31) / 32 * nc;
  for (int b = blockIdx.x; b < nt; b += gridDim.x) {
    const int i0 = b / nc * 32, t0 = b % nc * 64;
    if (tall) {
      __syncthreads();
      for (int q = threadIdx.x; q < 64 * 32; q += 256) {  // rows of G are columns of X
        const int t = t0 + q / 32, i = i0 + q % 32;
        tile[q / 32][q % 32] = t < p.l && i < p.s ? to_f(g[t * m.ldg + i]) : 0.f;
      }
      __syncthreads();
    }
#pragma unroll
    for (int q = threadIdx.x; q < 32 * 16; q += 256) {
      const int i = i0 + q / 16, t = t0 + q % 16 * 4;
      if (i >= p.s || t >= p.ldx) continue;
      f16x4_m h, lo;
      f32x4_m x;
      if (tall)
#pragma unroll
        for (int r = 0; r < 4; ++r) x[r] = tile[t - t0 + r][i - i0];
      else x = load4<T>(g + i * m.ldg + t, p.l - t);
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        f16_t v[2];
        split2(ldexpf(x[r], to) * rest, v);
        h[r] = v[0];
        lo[r] = v[1];
      }
      const long long o = (long long)i * p.ldx + t;
      *reinterpret_cast<f16x4_m*>(p.x + o) = h;
      *reinterpret_cast<f16x4_m*>(p.x + xp + o) = lo;
      if (t + 4 > p.l) {
        const f16x4_m z = {0, 0, 0, 0};  // values of the iterate itself come later
        *reinterpret_cast<f16x4_m*>(p.y + o) = z;
        *reinterpret_cast<f16x4_m*>(p.y + xp + o) = z;
      }
    }
  }
  const int pad = p.lda - p.s;
  for (long long q = (long long)blockIdx.x * 256 + threadIdx.x; q < (long long)pad * p.s; q += gridDim.x * 256LL) {
    const long long o = q / pad * p.lda + p.s + q % pad;
    p.a[o] = p.a[ap + o] = p.b[o] = p.b[ap + o] = 0;
  }
}

int up32(int v) { return (v + 31) / 32 * 32; }

struct PlaneLayout {
  long long bytes = 0, part = 0;
};
// planes of `n` matrices from `ws` on (null: the size alone), then the partial sums of the largest launch
PlaneLayout plane_layout(const int (*sl)[2], int n, char* ws, PlaneMat* out) {
  PlaneLayout w;
  PlaneShape gram[kJobs], poly[kJobs], step[kJobs];
  w.bytes = up256(kJobs * 4);
  for (int i = 0; i < n; ++i) {
    const int s = sl[i][0], l = sl[i][1], ldx = up32(l), lda = up32(s);
    const long long xb = up256((long long)s * ldx * 4), ab = up256((long long)s * lda * 4);
    if (out) {
      f16_t* at = reinterpret_cast<f16_t*>(ws + w.bytes);
      out[i] = {at, at + xb / 2, at + xb, at + xb + ab / 2, reinterpret_cast<int*>(ws) + i, s, l, lda, ldx};
    }
    w.bytes += 2 * xb + 2 * ab;
    gram[i] = {s, s, ldx};
    poly[i] = {s, s, lda};
    step[i] = {s, l, lda};
  }
  w.part = w.bytes;
  const long long f = std::max({plane_pick<2, true>(gram, n).part_floats, plane_pick<2, true>(poly, n).part_floats,
                                plane_pick<2, false>(step, n).part_floats});
  w.bytes += up256(f * 4);
  return w;
}

// `steps` >= 1 iterations on the matrices of l; the last one writes the results (dt) or the parameters (hyper)
template <typename T>
void plane_iterate(const MatList& l, int n, char* ws, int steps, int shift, const float* co, float eps, int dt,
                   const float* hyper, hipStream_t st) {
  PlaneMats pm;
  int sl[kJobs][2];
  long long most = 1;
  for (int i = 0; i < n; ++i) {
    sl[i][0] = std::min(l.m[i].rows, l.m[i].cols);
    sl[i][1] = std::max(l.m[i].rows, l.m[i].cols);
    most = std::max(most, (sl[i][0] + 31LL) / 32 * ((up32(sl[i][1]) + 63) / 64));
  }
  const PlaneLayout w = plane_layout(sl, n, ws, pm.p);
  float* part = reinterpret_cast<float*>(ws + w.part);
  launch(planes_kernel<T>, dim3((unsigned)std::min(most, 2048LL), n), dim3(256), 0, st, l, pm, eps);
  PlaneShape gram[kJobs], poly[kJobs], step[kJobs];
  PlaneJobs<GramEpi, kJobs> jg, jp;
  PlaneJobs<StepEpi, kJobs> js;
  jg.n = jp.n = js.n = n;
  for (int i = 0; i < n; ++i) {
    const PlaneMat& p = pm.p[i];
    gram[i] = {p.s, p.s, p.ldx};
    poly[i] = {p.s, p.s, p.lda};
    step[i] = {p.s, p.l, p.lda};
    const long long xp = (long long)p.s * p.ldx, ap = (long long)p.s * p.lda;
    jg.j[i] = {{p.x, p.ldx, xp}, {p.x, p.ldx, xp}, p.s, p.s, p.ldx, 0, 0, 0, 0, nullptr,
               {p.a, nullptr, p.lda, p.s, ap, kAs / (kXs * kXs), 0.f, p.expo, 0}};
    jp.j[i] = {{p.a, p.lda, ap}, {p.a, p.lda, ap}, p.s, p.s, p.lda, 0, 0, 0, 0, nullptr,
               {p.b, p.a, p.lda, p.s, ap, co[2] / kAs, co[1], nullptr, 0}};
    js.j[i] = {{p.b, p.lda, ap}, {p.x, p.ldx, xp}, p.s, p.l, p.s, 0, 0, 0, 0, nullptr,
               {p.y, p.x, xp, p.ldx, 0, 1.f / kAs, co[0], l.m[i].out, l.m[i].ldo, l.m[i].rows > l.m[i].cols,
                l.m[i].scale, hyper, p.expo, 0, 0}};
  }
  const PlanePick pg = plane_pick<2, true>(gram, n), pp = plane_pick<2, true>(poly, n), ps = plane_pick<2, false>(step, n);
  for (int k = 0; k < steps; ++k) {
    const bool last = k == steps - 1;
    for (int i = 0; i < n; ++i) {
      jg.j[i].e.drop = js.j[i].e.drop = k * shift;
      js.j[i].e.next = last ? INT_MAX : (k + 1) * shift;  // the result itself: no factor
      if (last) js.j[i].e.mode = hyper ? 4 : 1 + dt;
    }
    plane_run<f16_t, 2, false, false, true>(jg, pg, part, st);
    plane_run<f16_t, 2, false, false, true>(jp, pp, part, st);
    plane_run<f16_t, 2, false, true, false>(js, ps, part, st);
    for (int i = 0; i < n; ++i) {  // X and Y change places
      const f16_t* x = js.j[i].e.out;
      f16_t* y = const_cast<f16_t*>(js.j[i].e.in);
      js.j[i].e.out = y;
      js.j[i].e.in = x;
      js.j[i].b.p = jg.j[i].a.p = jg.j[i].b.p = x;
    }
  }
}

// --- matrices with a short side of up to 64: the whole step in one launch ---
// A block owns a slab of X, kCols columns of the long side (several in turn where there are more than kMaxSlabs),
// and keeps it in LDS through a step; what the blocks of a matrix share is the 64 x 64 Gram matrix, whose partial
// sums pass through memory between launches:
//   launch 0:  G -> planes (and the momentum update), partial G G^T
//   launch k:  A = sum of the partials, B = b A + c A A (every block for itself: 2 x 64^3), X <- a X + B X,
//              partial X X^T for the next launch; the last one writes the result or the parameter
// so five steps are six launches for up to kSlabMats matrices of any shapes, where the general products take
// seventeen and joins.  Bound by latency: a launch of 64 x 1728 is ~7.5 us, of which a fourth is the trip to the
// arguments, and about as much each the Gram partials, the step and the Gram product.  Measured, us, here / on planes:
// 16 x 343 49 / 68, 64 x 1728 53 / 98, 64 x 16384 103 / 139, 64 x 65536 182 / 213, four of these 250 / 417; a
// very long single one loses (16 x 200000 381 / 332).  kMaxSlabs 32 / 64 / 128: 64 x 16384 99 / 103 / 103, 64 x 65536
// 244 / 182 / 186, four of these 288 / 250 / 399.  G's planes are scaled by the power of two of the slab's largest value,
// and the norm is the trace of the partial Gram matrices, in 64 bits: no pass of its own.  Vectors' Adam rides on
// launch 0.
constexpr int kMaxSlabs = 64, kBatch = 16, kCols = 256, kSlab = 64 * kCols;
constexpr int kSlabThreads = 4 * kCols, kSlabWaves = kSlabThreads / 64;  // a wave: 16 columns, and one tile of a 64 x 64 matrix
static_assert(kSlabWaves == 16, "a wave for each tile of the Gram matrix");

struct SlabMat {
  const void* g;    // G, or the gradient
  void* out;        // the result, or the parameter
  float* mom;       // muon: momentum (vectors: first moment)
  float* sq;        // muon, vectors: second moment
  long long ldg, ldo;
  int rows, cols;   // rows 0: a vector of `count` values
  float scale;
  int nslab, sub;   // blocks, and slabs a block takes
  long long count;
  f16_t* x;         // planes, [slab][2][64][kCols], LDS order
  float* part;      // [2][nslab][64 * 64]
  float* expo;      // [nslab]: G = planes * 2^expo; [nslab] X's start exponent, a copy for each block
};
// matrices and vectors of a launch: as many as its arguments hold (4096 bytes, 320 of them for the rest), and a lane each
constexpr int kSlabMats = std::min<int>((4096 - 320) / (sizeof(SlabMat) + sizeof(int)), 64);
struct SlabList {
  int n, tick;  // tick: the last launch advances the step counter
  int start[kSlabMats + 1];
  SlabMat m[kSlabMats];
};

// place of 16-byte chunk c of row r: conflict-free for fragments along the row, two lanes a bank across it
__device__ __forceinline__ int slab_at(int r, int c) { return r * (kCols / 8) + (c ^ (r & 15)); }

// 16 x 16 tile (ti, tj) of M M^T over 32 W columns; M's planes: a slab's (SLAB), or of 64 x 64 in rows of 8 chunks
template <bool SLAB, int W>
__device__ __forceinline__ void gram_tile(const f16_t* m, int plane, int ti, int tj, int lane, f32x4_m& acc) {
  const auto frag = [&](int p, int row, int k) {
    const int r = row * 16 + (lane & 15), c = k * 4 + (lane >> 4);
    return *reinterpret_cast<const s16x8_v*>(m + p * plane + (SLAB ? slab_at(r, c) : r * 8 + (c ^ sw_kc<8>(r))) * 8);
  };
  f32x4_m c1 = {}, c2 = {};  // chains of their own
#pragma unroll
  for (int k = 0; k < W; ++k) {
    const s16x8_v a0 = frag(0, ti, k), a1 = frag(1, ti, k), b0 = frag(0, tj, k), b1 = frag(1, tj, k);
    c1 = plane_mfma(b1, a0, c1, f16_t());
    c2 = plane_mfma(b0, a1, c2, f16_t());
    acc = plane_mfma(b0, a0, acc, f16_t());
  }
  acc += c1 + c2;
}

// a thread's four neighbours u of a slab (row, and column within it): along the long side, or a tall matrix's short one
__device__ __forceinline__ int slab_i(bool tall, int u, int tid) {
  const int q = u * kSlabThreads + tid;
  return tall ? q % 16 * 4 : q / (kCols / 4);
}
__device__ __forceinline__ int slab_t(bool tall, int u, int tid) {
  const int q = u * kSlabThreads + tid;
  return tall ? q / 16 : q % (kCols / 4) * 4;
}
// PHASE 0: launch 0, 1: a step that is not the last, 2: the last
template <typename T, int PHASE>
__global__ __launch_bounds__(kSlabThreads) void slab_kernel(SlabList l, int k, int shift, float ca, float cb, float cc,
                                                            float eps, float* __restrict__ hyper) {
  __shared__ __align__(16) f16_t X[2 * kSlab];  // a wave's columns are its own: the step's result replaces them
  __shared__ __align__(16) f16_t A[2 * 64 * 64];
  __shared__ __align__(16) f16_t B[2 * 64 * 64];
  __shared__ double redd[kSlabWaves];
  __shared__ float redf[kSlabWaves];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  // this block's matrix: every lane looks at one start (the arguments are far away: one trip, not one per entry)
  const unsigned long long before = __ballot(lane < l.n && (int)blockIdx.x >= l.start[min(lane, kSlabMats)]);
  const int mi = __builtin_amdgcn_readfirstlane(__popcll(before) - 1);
  const SlabMat& m = l.m[mi];
  const int slab = blockIdx.x - l.start[mi];
  if (PHASE == 2 && hyper && l.tick && blockIdx.x == 0 && tid == 0) hyper[H_STEP] += 1.f;  // nothing of this launch reads it
  if (m.rows == 0) {
    if (PHASE == 0) {
      const float h[6] = {hyper[H_VLR], hyper[H_VB1], hyper[H_VB2], hyper[H_VEPS], 0.f, hyper[H_CLIP]};
      const AdamK ak = adam_k(h, hyper[H_STEP] + 1.f);
      for (long long q = slab * (long long)kSlabThreads + tid; q < m.count; q += m.nslab * (long long)kSlabThreads)
        adam_elem(ak, static_cast<float*>(m.out), static_cast<const float*>(m.g), m.mom, m.sq, q);
    }
    return;
  }
  const bool tall = m.rows > m.cols;
  const int s = min(m.rows, m.cols), len = max(m.rows, m.cols);
  f32x4_m gram = {};
  const int gi = wave >> 2, gj = wave & 3;  // this wave's tile of a 64 x 64 matrix
  f16_t* state = m.x + (long long)slab * m.sub * (2 * kSlab);

  if constexpr (PHASE == 0) {
    const float mu = hyper ? hyper[H_MU] : 0.f;
    const bool nest = hyper && hyper[H_NESTEROV] != 0.f;
    const T* g = static_cast<const T*>(m.g);
    // a thread: four neighbours in memory, four times; every load before the first store
    f32x4_m v[4];
    const auto load = [&](int b, bool keep) {
      const int t0 = (slab * m.sub + b) * kCols;
      f32x4_m w[4];
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        const int i = slab_i(tall, u, tid), t = t0 + slab_t(tall, u, tid);
        const int n = i < s && t < len ? (tall ? s - i : len - t) : 0;
        const long long o = tall ? t * m.ldg + i : i * m.ldg + t;
        v[u] = load4<T>(g + o, n);
        w[u] = hyper ? load4<float>(m.mom + o, n) : f32x4_m{0.f, 0.f, 0.f, 0.f};
      }
      if (!hyper) return;
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        const int i = slab_i(tall, u, tid), t = t0 + slab_t(tall, u, tid);
        const int n = i < s && t < len ? (tall ? s - i : len - t) : 0;
        w[u] += (1.f - mu) * (v[u] - w[u]);
        v[u] = nest ? v[u] + mu * (w[u] - v[u]) : w[u];
        if (keep) store4<float>(m.mom + (tall ? t * m.ldg + i : i * m.ldg + t), w[u], n);
      }
    };
    float big = 0.f;
    for (int b = 0; b < m.sub; ++b) {
      load(b, m.sub == 1);
#pragma unroll
      for (int u = 0; u < 16; ++u) big = fmaxf(big, fabsf(v[u >> 2][u & 3]));
    }
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) big = fmaxf(big, __shfl_xor(big, o, 64));
    if (lane == 0) redf[wave] = big;
    lds_barrier();
    big = redf[0];
#pragma unroll
    for (int w = 1; w < kSlabWaves; ++w) big = fmaxf(big, redf[w]);
    // values below 2^12; nothing to scale by where all are zero or some are not finite
    const int e = big > 0.f && big < __builtin_inff() ? ilogbf(big) + 1 - 12 : 0;
    if (tid == 0) m.expo[slab] = (float)e;
    for (int b = 0; b < m.sub; ++b) {
      if (m.sub > 1) load(b, true);
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        const int i = slab_i(tall, u, tid), t = slab_t(tall, u, tid);
        f16x4_m hi, lo;
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          f16_t p[2];
          split2(ldexpf(v[u][r], -e), p);
          hi[r] = p[0];
          lo[r] = p[1];
        }
        if (tall) {
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            const int o = slab_at(i + r, t >> 3) * 8 + (t & 7);
            X[o] = hi[r];
            X[kSlab + o] = lo[r];
          }
        } else {
          const int o = slab_at(i, t >> 3) * 8 + (t & 7);
          *reinterpret_cast<f16x4_m*>(X + o) = hi;
          *reinterpret_cast<f16x4_m*>(X + kSlab + o) = lo;
        }
      }
      lds_barrier();
#pragma unroll
      for (int u = 0; u < 4; ++u)
        reinterpret_cast<s16x8_v*>(state + (long long)b * (2 * kSlab))[u * kSlabThreads + tid] = reinterpret_cast<s16x8_v*>(X)[u * kSlabThreads + tid];
      if (gi >= gj) gram_tile<true, kCols / 32>(X, kSlab, gi, gj, lane, gram);
      lds_barrier();
    }
  } else {
    s16x8_v xr[4];  // the slab is on its way while the Gram matrix is put together
#pragma unroll
    for (int u = 0; u < 4; ++u) xr[u] = reinterpret_cast<const s16x8_v*>(state)[u * kSlabThreads + tid];
    // A: a thread adds four neighbours of a row over the slabs, in their order.  What lies beyond the short side is
    // zero and is not read; the loads of kBatch slabs are in flight together
    const float* part = m.part + (long long)((k - 1) & 1) * m.nslab * 4096 + tid * 4;
    const int ri = tid >> 4, rj = (tid & 15) * 4;
    const bool some = ri < s && rj < s;
    f32x4_m sum = {};
    float alpha = 1.f / kAs, beta = ca;
    int ex;  // of the result beside alpha and beta
    const int start = k > 1 ? (int)m.expo[m.nslab + slab] : 0;
    const auto slabs = [&](auto f) {
      for (int z0 = 0; z0 < m.nslab; z0 += kBatch) {
        f32x4_m p[kBatch];
#pragma unroll
        for (int z = 0; z < kBatch; ++z) {
          p[z] = f32x4_m{0.f, 0.f, 0.f, 0.f};
          if (some && z0 + z < m.nslab) p[z] = *reinterpret_cast<const f32x4_m*>(part + (long long)(z0 + z) * 4096);
        }
#pragma unroll
        for (int z = 0; z < kBatch; ++z) f(min(z0 + z, m.nslab - 1), p[z]);
      }
    };
    if (k == 1) {
      double d[4] = {};
      slabs([&](int z, const f32x4_m& p) {
        const double f = ldexp(1.0, 2 * (int)m.expo[z]);
#pragma unroll
        for (int r = 0; r < 4; ++r) d[r] += f * p[r];
      });
      double tr = 0.;
#pragma unroll
      for (int r = 0; r < 4; ++r)
        if (rj + r == ri) tr = d[r];
      tr = wave_sum_d(tr);
      if (lane == 0) redd[wave] = tr;
      lds_barrier();
      tr = 0.;
#pragma unroll
      for (int w = 0; w < kSlabWaves; ++w) tr += redd[w];
      const double size = sqrt(tr), inv = 1. / (size + (double)eps);
#pragma unroll
      for (int r = 0; r < 4; ++r) sum[r] = (float)(d[r] * inv * inv);
      const int e = start_exponent(size * inv);
      if (tid == 0) m.expo[m.nslab + slab] = (float)e;
      // from G's planes to X's, exponent and the rest apart (a slab of zeros may have any)
      const float r0 = (float)frexp(kXs * inv, &ex);
      ex += (int)m.expo[slab] + (PHASE == 2 ? 0 : max(e - shift, 0));
      alpha *= r0;
      beta *= r0;
    } else {
      slabs([&](int, const f32x4_m& p) { sum += p; });
      const int in = max(start - (k - 1) * shift, 0);
#pragma unroll
      for (int r = 0; r < 4; ++r) sum[r] = ldexpf(sum[r] * (1.f / (kXs * kXs)), -2 * in);
      ex = (PHASE == 2 ? 0 : max(start - k * shift, 0)) - in;
    }
    {
      f16x4_m hi, lo;
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        f16_t q[2];
        split2(sum[r] * kAs, q);
        hi[r] = q[0];
        lo[r] = q[1];
      }
      const int o = (ri * 8 + ((rj >> 3) ^ sw_kc<8>(ri))) * 8 + (rj & 7);
      *reinterpret_cast<f16x4_m*>(A + o) = hi;
      *reinterpret_cast<f16x4_m*>(A + 64 * 64 + o) = lo;
    }
    lds_barrier();
    f32x4_m sqr = {};
    gram_tile<false, 2>(A, 64 * 64, gi, gj, lane, sqr);
    {
      const int i = gi * 16 + (lane & 15), j = gj * 16 + (lane >> 4) * 4;
      const int o = (i * 8 + ((j >> 3) ^ sw_kc<8>(i))) * 8 + (j & 7);
      const f16x4_m h = *reinterpret_cast<const f16x4_m*>(A + o), lw = *reinterpret_cast<const f16x4_m*>(A + 64 * 64 + o);
      f16x4_m oh, ol;
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        f16_t q[2];
        split2(cc / kAs * sqr[r] + cb * ((float)h[r] + (float)lw[r]), q);
        oh[r] = q[0];
        ol[r] = q[1];
      }
      *reinterpret_cast<f16x4_m*>(B + o) = oh;
      *reinterpret_cast<f16x4_m*>(B + 64 * 64 + o) = ol;
    }
    for (int b = 0; b < m.sub; ++b) {
      if (b > 0) {
#pragma unroll
        for (int u = 0; u < 4; ++u) xr[u] = reinterpret_cast<const s16x8_v*>(state + (long long)b * (2 * kSlab))[u * kSlabThreads + tid];
      }
#pragma unroll
      for (int u = 0; u < 4; ++u) reinterpret_cast<s16x8_v*>(X)[u * kSlabThreads + tid] = xr[u];
      lds_barrier();
      // a wave: 16 columns, all 64 rows
      f32x4_m acc[4] = {};
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        s16x8_v fx[2];
#pragma unroll
        for (int p = 0; p < 2; ++p) {
          const int kr = h * 32 + 8 * (lane >> 4) + ((lane & 15) >> 2), c = wave * 2 + ((lane & 3) >> 1);
          typedef __attribute__((address_space(3))) s16x4_v* lp;
          const f16_t* base = X + p * kSlab + (lane & 1) * 4;
          const s16x4_v lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lp)(base + slab_at(kr, c) * 8));
          const s16x4_v hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lp)(base + slab_at(kr + 4, c) * 8));
          fx[p] = __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
        }
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          const int r = q * 16 + (lane & 15), o = (r * 8 + ((h * 4 + (lane >> 4)) ^ sw_kc<8>(r))) * 8;
          const s16x8_v b0 = *reinterpret_cast<const s16x8_v*>(B + o), b1 = *reinterpret_cast<const s16x8_v*>(B + 64 * 64 + o);
          acc[q] = plane_mfma(fx[1], b0, acc[q], f16_t());
          acc[q] = plane_mfma(fx[0], b1, acc[q], f16_t());
          acc[q] = plane_mfma(fx[0], b0, acc[q], f16_t());
        }
      }
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const int i = q * 16 + (lane & 15), t = wave * 16 + (lane >> 4) * 4;
        const int o = slab_at(i, t >> 3) * 8 + (t & 7);
        const f16x4_m h = *reinterpret_cast<const f16x4_m*>(X + o), lw = *reinterpret_cast<const f16x4_m*>(X + kSlab + o);
        f32x4_m x;
#pragma unroll
        for (int r = 0; r < 4; ++r) x[r] = ldexpf(alpha * acc[q][r] + beta * ((float)h[r] + (float)lw[r]), ex);
        if constexpr (PHASE == 1) {
          f16x4_m oh, ol;
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            f16_t p[2];
            split2(x[r], p);
            oh[r] = p[0];
            ol[r] = p[1];
          }
          *reinterpret_cast<f16x4_m*>(X + o) = oh;
          *reinterpret_cast<f16x4_m*>(X + kSlab + o) = ol;
        } else {  // the two planes' places hold one f32: its high half and its low half
          f16x4_m oh, ol;
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            const unsigned w = __float_as_uint(x[r] * (1.f / kXs));
            oh[r] = __builtin_bit_cast(f16_t, (unsigned short)(w >> 16));
            ol[r] = __builtin_bit_cast(f16_t, (unsigned short)w);
          }
          *reinterpret_cast<f16x4_m*>(X + o) = oh;
          *reinterpret_cast<f16x4_m*>(X + kSlab + o) = ol;
        }
      }
      lds_barrier();
      if constexpr (PHASE == 1) {
#pragma unroll
        for (int u = 0; u < 4; ++u)
          reinterpret_cast<s16x8_v*>(state + (long long)b * (2 * kSlab))[u * kSlabThreads + tid] = reinterpret_cast<s16x8_v*>(X)[u * kSlabThreads + tid];
        if (gi >= gj) gram_tile<true, kCols / 32>(X, kSlab, gi, gj, lane, gram);
        lds_barrier();
      } else {
        const int t0 = (slab * m.sub + b) * kCols;
        const float lr = hyper ? hyper[H_LR] : 0.f, clip = hyper ? hyper[H_CLIP] : 0.f;
        const float keep = hyper ? 1.f - lr * hyper[H_WD] : 0.f, rate = lr * m.scale;
        f32x4_m w[4];
#pragma unroll
        for (int u = 0; u < 4; ++u) {
          const int i = slab_i(tall, u, tid), t = t0 + slab_t(tall, u, tid);
          const int n = hyper && i < s && t < len ? (tall ? s - i : len - t) : 0;
          w[u] = load4<float>(static_cast<const float*>(m.out) + (tall ? t * m.ldo + i : i * m.ldo + t), n);
        }
#pragma unroll
        for (int u = 0; u < 4; ++u) {
          const int i = slab_i(tall, u, tid), t = slab_t(tall, u, tid);
          const int n = i < s && t0 + t < len ? (tall ? s - i : len - t0 - t) : 0;
          const long long o = tall ? (t0 + t) * m.ldo + i : i * m.ldo + t0 + t;
          f32x4_m x;
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            const int at = tall ? slab_at(i + r, t >> 3) * 8 + (t & 7) : slab_at(i, t >> 3) * 8 + (t & 7) + r;
            x[r] = __uint_as_float((unsigned)__builtin_bit_cast(unsigned short, X[at]) << 16 |
                                   __builtin_bit_cast(unsigned short, X[kSlab + at]));
          }
          if (hyper) {
            x = w[u] * keep - rate * x;
            if (clip > 0.f)
#pragma unroll
              for (int r = 0; r < 4; ++r) x[r] = fminf(fmaxf(x[r], -clip), clip);
            store4<float>(static_cast<float*>(m.out) + o, x, n);
          } else {
            store4<T>(static_cast<T*>(m.out) + o, x, n);
          }
        }
        lds_barrier();
      }
    }
  }
  if constexpr (PHASE != 2) {
    if (gi < gj) return;  // the upper triangle is the lower one's mirror
    float* part = m.part + ((long long)(k & 1) * m.nslab + slab) * 4096;
    const int i = gi * 16 + (lane & 15), j = gj * 16 + (lane >> 4) * 4;
    *reinterpret_cast<f32x4_m*>(part + i * 64 + j) = gram;
    if (gi > gj)
#pragma unroll
      for (int r = 0; r < 4; ++r) part[(j + r) * 64 + i] = gram[r];
  }
}

bool slab_takes(long long rows, long long cols) { return std::min(rows, cols) <= 64; }

// blocks of a matrix, and its part of the workspace from `ws` on
long long slab_place(SlabMat& m, char* ws) {
  const int len = std::max(m.rows, m.cols), all = (len + kCols - 1) / kCols;
  m.sub = (all + kMaxSlabs - 1) / kMaxSlabs;
  m.nslab = (all + m.sub - 1) / m.sub;
  const long long xb = (long long)m.nslab * m.sub * kSlab * 4, pb = 2LL * m.nslab * 4096 * 4;
  m.x = reinterpret_cast<f16_t*>(ws);
  m.part = reinterpret_cast<float*>(ws + xb);
  m.expo = reinterpret_cast<float*>(ws + xb + pb);
  return xb + pb + up256(2 * m.nslab * 4);
}

// one launch and one per step; `hyper`: the Muon step of the list (f32)
template <typename T>
void slab_run(SlabList& l, int steps, int shift, const float* co, float eps, float* hyper, hipStream_t st) {
  int at = 0;
  for (int i = 0; i < l.n; ++i) {
    l.start[i] = at;
    at += l.m[i].nslab;
  }
  launch(slab_kernel<T, 0>, dim3(at), dim3(kSlabThreads), 0, st, l, 0, shift, co[0], co[1], co[2], eps, hyper);
  for (int k = 1; k < steps; ++k)
    launch(slab_kernel<T, 1>, dim3(at), dim3(kSlabThreads), 0, st, l, k, shift, co[0], co[1], co[2], eps, hyper);
  launch(slab_kernel<T, 2>, dim3(at), dim3(kSlabThreads), 0, st, l, steps, shift, co[0], co[1], co[2], eps, hyper);
}

// Whether iterates that start within |X| <= 1 stay where the planes hold them: |X| < 2^16 / kXs, |A| and |B|
// (largest entry <= largest singular value) < 2^16 / kAs.  *shift: a step makes no singular value larger by more than
// 2^shift.  The polynomial at 512 points (7 us of a call's host time), with a margin for what lies between them: its second
// derivative is below 26 * 60 / r where the first test holds, so at most 1e-3 r above its neighbours
bool planes_hold(int steps, const float* co, int* shift) {
  if (steps < 1) return false;
  double r = 1.0, gain = std::fabs(co[0]);
  for (int k = 0; k < steps; ++k) {
    if (r > 7.5 || std::fabs(co[1]) * r * r + std::fabs(co[2]) * r * r * r * r > 60.) return false;
    double next = 0;
    for (int q = 1; q <= 512; ++q) {
      const double x = r * q / 512, x2 = x * x, g = std::fabs(co[0] + x2 * (co[1] + x2 * co[2]));
      gain = std::max(gain, g);
      next = std::max(next, x * g);
    }
    r = next * 1.01 + 1e-3 * r;
  }
  *shift = std::max(0, std::ilogb(gain * 1.01) + 1);
  return r <= 7.5;
}

__global__ void muon_tick_kernel(float* hyper) { hyper[H_STEP] += 1.f; }

struct Layout {
  long long part, u, x, x2, a, b, mat, total;
};
// Every matrix has its own partial sums and (muon) its own update.  Behind them one region, either for the
// planes of up to kJobs matrices at a time (`planes`) or, with the f32 products, for one matrix after the
// other.
void size_mat(Layout& w, long long rows, long long cols) {
  const long long s = std::min(rows, cols), l = std::max(rows, cols);
  w.x = std::max(w.x, up256(s * l * 4));
  w.a = std::max(w.a, up256(s * s * 4));
  w.mat = std::max({w.mat, mat_f32_ws_bytes(s, s, l), mat_f32_ws_bytes(s, s, s), mat_f32_ws_bytes(s, l, s)});
}
void place(Layout& w, long long nmat, long long ubytes, long long planes) {
  const long long x = w.x, a = w.a, m = w.mat;
  w.part = 0;
  w.u = up256(nmat * kNormBlocks * 8);
  w.x = w.u + up256(ubytes);
  w.x2 = w.x + x;
  w.a = w.x2 + x;
  w.b = w.a + a;
  w.mat = w.b + a;
  w.total = std::max(w.mat + m, w.x + planes);
}

// bytes of the largest group of kJobs matrices, in the order the runs take them; rc(i): rows and cols of
// matrix i (empty ones are left out)
template <class F> long long plane_bytes(int n, F rc) {
  int sl[kJobs][2], at = 0;
  long long most = 0;
  for (int i = 0; i <= n; ++i) {
    long long r = 0, c = 0;
    if (i < n) rc(i, r, c);
    if (r * c > 0 && !slab_takes(r, c)) {
      sl[at][0] = (int)std::min(r, c);
      sl[at][1] = (int)std::max(r, c);
      ++at;
    }
    if (at == kJobs || (i == n && at > 0)) {
      most = std::max(most, plane_layout(sl, at, nullptr, nullptr).bytes);
      at = 0;
    }
  }
  return most;
}

// the same of the largest group of kSlabMats matrices with a short side for slab_kernel
template <class F> long long slab_bytes(int n, F rc) {
  long long most = 0, sum = 0;
  int at = 0;
  for (int i = 0; i < n; ++i) {
    long long r = 0, c = 0;
    rc(i, r, c);
    if (r * c == 0 || !slab_takes(r, c)) continue;
    SlabMat m = {};
    m.rows = (int)r;
    m.cols = (int)c;
    sum += slab_place(m, nullptr);
    most = std::max(most, sum);
    if (++at == kSlabMats) at = 0, sum = 0;
  }
  return most;
}

// `steps` iterations on m.x; returns where the result is
float* iterate(const Mat& m, const Layout& w, char* ws, int steps, const float* co, hipStream_t st) {
  const long long s = std::min(m.rows, m.cols), l = std::max(m.rows, m.cols);
  float* x = m.x;
  float* y = reinterpret_cast<float*>(ws + w.x2);
  float* A = reinterpret_cast<float*>(ws + w.a);
  float* B = reinterpret_cast<float*>(ws + w.b);
  for (int k = 0; k < steps; ++k) {
    MatArgs p = {};
    p.a = p.b = x; p.lda = p.ldb = l;
    p.I = p.J = s; p.K = l;
    p.e.out = A; p.e.ldo = s; p.e.alpha = 1.f;
    mat_f32(false, false, p, ws + w.mat, st);
    p.a = p.b = A; p.lda = p.ldb = s;  // A is symmetric: A A = A A^T
    p.K = s;
    p.e.out = B; p.e.alpha = co[2];
    p.e.residual = A; p.e.ldr = s; p.e.beta = co[1];
    mat_f32(false, false, p, ws + w.mat, st);
    p.a = B; p.b = x; p.ldb = l;
    p.J = l;
    p.e.out = y; p.e.ldo = l; p.e.alpha = 1.f;
    p.e.residual = x; p.e.ldr = l; p.e.beta = co[0];
    mat_f32(false, true, p, ws + w.mat, st);
    std::swap(x, y);
  }
  return x;
}

const char* ns_check(int steps, const float* co, float eps) {
  if (steps < 0 || steps > 64) return "steps must be 0..64";
  if (!co || !std::isfinite(co[0]) || !std::isfinite(co[1]) || !std::isfinite(co[2])) return "three finite coefficients needed";
  if (!(eps >= 0.f) || !std::isfinite(eps)) return "eps must be finite and not negative";
  return nullptr;
}

const char* mats_check(const cgan3d_ortho_mat* m, int n, int dt) {
  if (n < 0 || (n > 0 && !m)) return "null list";
  if (dt < CGAN3D_DT_F32 || dt > CGAN3D_DT_F16) return "unknown dtype";
  for (int i = 0; i < n; ++i) {
    if (m[i].rows < 0 || m[i].cols < 0 || m[i].rows > 1 << 30 || m[i].cols > 1 << 30) return "negative or too large size";
    if ((long long)m[i].rows * m[i].cols == 0) continue;
    if (!m[i].g || !m[i].out) return "null matrix";
    if (m[i].ldg < m[i].cols || m[i].ldo < m[i].cols) return "row stride smaller than the row";
    const long long t = (std::max(m[i].rows, m[i].cols) + 63LL) / 64, u = (std::min(m[i].rows, m[i].cols) + 63LL) / 64;
    if (t * u > INT_MAX) return "matrix too large for one launch";
  }
  return nullptr;
}

// The f32 products run on tiles of 64 x 64, 256 threads each: HIP takes fewer than 2^32 threads.  (On planes the largest
// matrices that fit the memory stay below it.)
bool mat_grid_holds(long long rows, long long cols) { return ((rows + 63) / 64) * ((cols + 63) / 64) < 1 << 24; }

Layout ortho_layout(const cgan3d_ortho_mat* m, int n) {
  Layout w = {};
  for (int i = 0; i < n; ++i) size_mat(w, m[i].rows, m[i].cols);
  const auto rc = [&](int i, long long& r, long long& c) { r = m[i].rows; c = m[i].cols; };
  place(w, n, 0, std::max(plane_bytes(n, rc), slab_bytes(n, rc)));
  return w;
}

template <typename T>
void ortho_run(const cgan3d_ortho_mat* mats, int n, int dt, const Layout& w, char* ws, int steps, const float* co,
               float eps, hipStream_t st) {
  int shift = 0;
  const bool planes = planes_hold(steps, co, &shift);
  if (planes) {
    SlabList sl = {};
    long long used = 0;
    for (int i = 0; i < n; ++i) {
      const cgan3d_ortho_mat& q = mats[i];
      if ((long long)q.rows * q.cols > 0 && slab_takes(q.rows, q.cols)) {
        SlabMat& m = sl.m[sl.n++];
        m = {};
        m.g = q.g; m.out = q.out; m.ldg = q.ldg; m.ldo = q.ldo; m.rows = q.rows; m.cols = q.cols;
        used += slab_place(m, ws + w.x + used);
      }
      if (sl.n == kSlabMats || (i == n - 1 && sl.n > 0)) {
        slab_run<T>(sl, steps, shift, co, eps, nullptr, st);
        sl.n = 0;
        used = 0;
      }
    }
  }
  MatList l;
  int at = 0;
  const auto flush = [&]() {
    if (!at) return;
    launch(norm_kernel<T>, dim3(kNormBlocks, at), dim3(256), 0, st, l);
    if (planes) {
      plane_iterate<T>(l, at, ws + w.x, steps, shift, co, eps, dt, nullptr, st);
    } else {
      const unsigned blocks = (unsigned)std::min(((long long)l.m[0].rows * l.m[0].cols + 1023) / 1024, 4096LL);
      launch(scale_kernel<T>, dim3(blocks, 1), dim3(256), 0, st, l, eps);
      l.m[0].x = iterate(l.m[0], w, ws, steps, co, st);
      launch(ortho_out_kernel<T>, dim3(blocks, 1), dim3(256), 0, st, l);
    }
    at = 0;
  };
  for (int i = 0; i < n; ++i) {
    const cgan3d_ortho_mat& q = mats[i];
    if ((long long)q.rows * q.cols == 0 || (planes && slab_takes(q.rows, q.cols))) continue;
    l.m[at++] = {q.g, q.out, q.ldg, q.ldo, q.rows, q.cols, 1.f, reinterpret_cast<float*>(ws + w.x),
                 reinterpret_cast<double*>(ws + w.part) + (long long)i * kNormBlocks};
    if (at == (planes ? kJobs : 1)) flush();
  }
  flush();
}

const char* segs_check(const cgan3d_muon_seg* s, int n) {
  if (n < 0 || (n > 0 && !s)) return "null list";
  for (int i = 0; i < n; ++i) {
    if (s[i].offset < 0 || s[i].rows < 0 || s[i].cols < 0 || s[i].rows > 1 << 30) return "negative or too large size";
    if (s[i].rows > 0 && s[i].cols > 1 << 30) return "negative or too large size";
    if (s[i].rows > 0) {
      const long long t = (std::max(s[i].rows, s[i].cols) + 63) / 64, u = (std::min(s[i].rows, s[i].cols) + 63) / 64;
      if (t * u > INT_MAX) return "matrix too large for one launch";
    }
  }
  return nullptr;
}

Layout muon_layout(const cgan3d_muon_seg* s, int n) {
  Layout w = {};
  long long nm = 0, u = 0;
  for (int i = 0; i < n; ++i)
    if (s[i].rows > 0) {
      size_mat(w, s[i].rows, s[i].cols);
      u += up256(s[i].rows * s[i].cols * 4);
      ++nm;
    }
  const auto rc = [&](int i, long long& r, long long& c) { r = s[i].rows; c = s[i].cols; };
  place(w, nm, u, std::max(plane_bytes(n, rc), slab_bytes(n, rc)));
  return w;
}

}  // namespace
}  // namespace cg

using namespace cg;

extern "C" int64_t cgan3d_orthogonalize_ws_bytes(const cgan3d_ortho_mat* mats, int32_t n, int32_t dtype) {
  if (const char* e = mats_check(mats, n, dtype)) {
    set_error("cgan3d_orthogonalize_ws_bytes: %s", e);
    return -1;
  }
  return ortho_layout(mats, n).total;
}

extern "C" int cgan3d_orthogonalize(const cgan3d_ortho_mat* mats, int32_t n, int32_t dtype, int32_t steps,
                                    const float* coefficients, float eps, void* ws, int64_t ws_bytes,
                                    void* stream) try {
  const char* e = mats_check(mats, n, dtype);
  CG_CHECK_ARG(!e, "cgan3d_orthogonalize: %s", e);
  e = ns_check(steps, coefficients, eps);
  CG_CHECK_ARG(!e, "cgan3d_orthogonalize: %s", e);
  int shift = 0;
  if (!planes_hold(steps, coefficients, &shift))
    for (int i = 0; i < n; ++i)
      CG_CHECK_ARG(mat_grid_holds(mats[i].rows, mats[i].cols), "cgan3d_orthogonalize: matrix too large for one launch");
  const Layout w = ortho_layout(mats, n);
  CG_CHECK_ARG(ws_bytes >= w.total && (w.total == 0 || (ws && reinterpret_cast<uintptr_t>(ws) % 16 == 0)),
               "cgan3d_orthogonalize: workspace of %lld bytes (16-byte aligned) needed, got %lld", w.total,
               (long long)ws_bytes);
  hipStream_t st = (hipStream_t)stream;
  char* base = static_cast<char*>(ws);
  if (dtype == CGAN3D_DT_F32) ortho_run<float>(mats, n, dtype, w, base, steps, coefficients, eps, st);
  else if (dtype == CGAN3D_DT_BF16) ortho_run<bf16_t>(mats, n, dtype, w, base, steps, coefficients, eps, st);
  else ortho_run<f16_t>(mats, n, dtype, w, base, steps, coefficients, eps, st);
  CG_LAUNCH_CHECK("cgan3d_orthogonalize");
  return CGAN3D_OK;
} catch (...) {
  set_error("cgan3d_orthogonalize: out of host memory");
  return CGAN3D_EHIP;
}

extern "C" int64_t cgan3d_muon_ws_bytes(const cgan3d_muon_seg* segs, int32_t n) {
  if (const char* e = segs_check(segs, n)) {
    set_error("cgan3d_muon_ws_bytes: %s", e);
    return -1;
  }
  return muon_layout(segs, n).total;
}

extern "C" int cgan3d_muon_step(float* param, const float* grad, float* momentum, float* exp_avg_sq,
                                const cgan3d_muon_seg* segs, int32_t n, float* hyper, int32_t steps,
                                const float* coefficients, float eps, void* ws, int64_t ws_bytes, void* stream) try {
  const char* e = segs_check(segs, n);
  CG_CHECK_ARG(!e, "cgan3d_muon_step: %s", e);
  e = ns_check(steps, coefficients, eps);
  CG_CHECK_ARG(!e, "cgan3d_muon_step: %s", e);
  CG_CHECK_ARG(param && grad && momentum && exp_avg_sq && hyper, "cgan3d_muon_step: null operand");
  int shift = 0;
  const bool planes = planes_hold(steps, coefficients, &shift);
  for (int i = 0; i < n && !planes; ++i)
    CG_CHECK_ARG(segs[i].rows == 0 || mat_grid_holds(segs[i].rows, segs[i].cols),
                 "cgan3d_muon_step: matrix too large for one launch");
  const Layout w = muon_layout(segs, n);
  CG_CHECK_ARG(ws_bytes >= w.total && (w.total == 0 || (ws && reinterpret_cast<uintptr_t>(ws) % 16 == 0)),
               "cgan3d_muon_step: workspace of %lld bytes (16-byte aligned) needed, got %lld", w.total,
               (long long)ws_bytes);
  hipStream_t st = (hipStream_t)stream;
  char* base = static_cast<char*>(ws);
  float* u = reinterpret_cast<float*>(base + w.u);
  double* part = reinterpret_cast<double*>(base + w.part);
  // segment i: a matrix of slab_kernel, another one, or a vector; vectors ride along with the first list of the
  // former as long as there is room
  const auto is_slab = [&](int i) { return planes && segs[i].rows > 0 && segs[i].cols > 0 && slab_takes(segs[i].rows, segs[i].cols); };
  int slabs = 0;
  for (int i = 0; i < n; ++i) slabs += is_slab(i);
  int room = slabs > 0 ? kSlabMats - std::min(slabs, kSlabMats) : 0;
  const int rides = room;
  long long uo = 0;
  int nm = 0, at = 0;
  SegList l;
  const auto flush = [&]() {
    if (at > 0)
      launch(muon_moment_kernel, dim3(kNormBlocks, at), dim3(256), 0, st, l, param, grad, momentum, exp_avg_sq,
             (const float*)hyper, u, part);
    at = 0;
  };
  for (int i = 0; i < n; ++i) {
    const long long total = segs[i].rows > 0 ? segs[i].rows * segs[i].cols : segs[i].cols;
    if (!total || is_slab(i)) continue;
    if (segs[i].rows > 0) {
      l.mat[at] = nm++;
      l.u[at] = uo / 4;
      uo += up256(total * 4);
    } else {
      if (room > 0) {
        --room;
        continue;
      }
      l.mat[at] = -1;
    }
    l.s[at] = segs[i];
    if (++at == kList) flush();
  }
  flush();
  uo = 0;
  nm = 0;
  MatList q;
  int qn = 0;
  const auto run = [&]() {
    if (!qn) return;
    if (planes) {
      plane_iterate<float>(q, qn, base + w.x, steps, shift, coefficients, eps, 0, hyper, st);
    } else {
      const unsigned blocks = (unsigned)std::min(((long long)q.m[0].rows * q.m[0].cols + 1023) / 1024, 4096LL);
      launch(scale_kernel<float>, dim3(blocks, 1), dim3(256), 0, st, q, eps);
      q.m[0].x = iterate(q.m[0], w, base, steps, coefficients, st);
      launch(muon_apply_kernel, dim3(blocks, 1), dim3(256), 0, st, q, (const float*)hyper);
    }
    qn = 0;
  };
  for (int i = 0; i < n; ++i) {
    const long long total = segs[i].rows * segs[i].cols;
    if (segs[i].rows == 0 || !total || is_slab(i)) continue;
    q.m[qn] = {u + uo / 4, param + segs[i].offset, segs[i].cols, segs[i].cols, (int)segs[i].rows, (int)segs[i].cols,
               segs[i].lr_scale, reinterpret_cast<float*>(base + w.x), part + (long long)nm * kNormBlocks};
    ++nm;
    uo += up256(total * 4);
    if (++qn == (planes ? kJobs : 1)) run();
  }
  run();
  SlabList sl = {};
  long long used = 0;
  int left = slabs, ride = rides;
  for (int i = 0; i < n && left > 0; ++i) {
    if (!is_slab(i)) continue;
    SlabMat& m = sl.m[sl.n++];
    m = {};
    m.g = grad + segs[i].offset; m.out = param + segs[i].offset; m.mom = momentum + segs[i].offset;
    m.rows = (int)segs[i].rows; m.cols = (int)segs[i].cols;
    m.ldg = m.ldo = m.cols;
    m.scale = segs[i].lr_scale;
    used += slab_place(m, base + w.x + used);
    if (--left > 0 && sl.n < kSlabMats) continue;
    for (int v = 0; v < n && ride > 0; ++v) {
      if (segs[v].rows > 0 || segs[v].cols == 0) continue;
      SlabMat& x = sl.m[sl.n++];
      x = {};
      x.g = grad + segs[v].offset; x.out = param + segs[v].offset; x.mom = momentum + segs[v].offset;
      x.sq = exp_avg_sq + segs[v].offset;
      x.count = segs[v].cols;
      x.nslab = (int)std::max(1LL, std::min((x.count + 4095) / 4096, 256LL));
      --ride;
    }
    ride = 0;
    sl.tick = left == 0;
    slab_run<float>(sl, steps, shift, coefficients, eps, hyper, st);
    sl.n = 0;
    used = 0;
  }
  if (slabs == 0) launch(muon_tick_kernel, dim3(1), dim3(1), 0, st, hyper);
  CG_LAUNCH_CHECK("cgan3d_muon_step");
  return CGAN3D_OK;
} catch (...) {
  set_error("cgan3d_muon_step: out of host memory");
  return CGAN3D_EHIP;
}
