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
  if ((m.ldg == m.cols || m.rows == 1) && (reinterpret_cast<uintptr_t>(g) & 15) == 0) {
    for (long long q = tid; q < total / V; q += kNormBlocks * 256LL) {
      const vecT x = reinterpret_cast<const vecT*>(g)[q];
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

template <typename T>
__global__ __launch_bounds__(256) void scale_kernel(MatList l, float eps) {
  const Mat& m = l.m[blockIdx.y];
  const double s = block_sum_d(m.part[threadIdx.x]);  // one partial sum a thread
  const float norm = (float)(sqrt(s) + (double)eps);
  const T* g = static_cast<const T*>(m.g);
  const bool tall = m.rows > m.cols;
  const int lng = tall ? m.rows : m.cols;
  const long long total = (long long)m.rows * m.cols;
  for (long long q = (long long)blockIdx.x * 256 + threadIdx.x; q < total; q += gridDim.x * 256LL) {
    const long long i = q / lng, t = q - i * lng;
    m.x[q] = to_f(tall ? g[t * m.ldg + i] : g[i * m.ldg + t]) / norm;
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
  // called by whole waves: lane l has row l % 16 and columns 4 (l / 16) .. + 3 of a 16 x 16 block
  __device__ __forceinline__ void put(int i, int j, f32x4_m v, int jn, bool mirror) const {
    const long long o = (long long)i * ld + j;
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

  __device__ __forceinline__ bool turned() const { return tall && mode; }

  // four values at p, neighbours in memory, n of them
  template <typename T> static __device__ __forceinline__ void store(T* p, f32x4_m x, int n) {
    typedef T v4 __attribute__((ext_vector_type(4)));
    if (n >= 4 && (reinterpret_cast<uintptr_t>(p) & (4 * sizeof(T) - 1)) == 0) {
      v4 o;
#pragma unroll
      for (int r = 0; r < 4; ++r) o[r] = (T)x[r];
      *reinterpret_cast<v4*>(p) = o;
    } else {
#pragma unroll
      for (int r = 0; r < 4; ++r)
        if (r < n) p[r] = (T)x[r];
    }
  }
  // the last step's values x at offset d of the result or the parameter, n of them
  __device__ __forceinline__ void finish(long long d, f32x4_m x, int n) const {
    x *= 1.f / kXs;
    if (mode == 1 + CGAN3D_DT_F32) {
      store(static_cast<float*>(res) + d, x, n);
    } else if (mode == 1 + CGAN3D_DT_BF16) {
      store(static_cast<bf16_t*>(res) + d, x, n);
    } else if (mode == 1 + CGAN3D_DT_F16) {
      store(static_cast<f16_t*>(res) + d, x, n);
    } else {
      float* p = static_cast<float*>(res) + d;
      const float lr = hyper[H_LR], clip = hyper[H_CLIP], keep = 1.f - lr * hyper[H_WD], rate = lr * scale;
      f32x4_m w;
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        w[r] = r < n ? p[r] * keep - rate * x[r] : 0.f;
        if (clip > 0.f) w[r] = fminf(fmaxf(w[r], -clip), clip);
      }
      store(p, w, n);
    }
  }
  // four columns from j of rows i, i + STEP, .. + 3 STEP: every load before the first store
  template <int STEP> __device__ __forceinline__ void put4(int i, int j, f32x4_m* v, int I, int jn) const {
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
      for (int r = 0; r < 4; ++r) v[u][r] = alpha * v[u][r] + beta * ((float)a[u][r] + (float)c[u][r]);
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
  __device__ __forceinline__ void put(int i, int j, f32x4_m v, int jn, bool) const {
    f32x4_m w[4] = {v};
    put4<1>(i, j, w, i + 1, jn);
    if (turned())
#pragma unroll
      for (int r = 0; r < 4; ++r)
        if (r < jn) finish((j + r) * ldr + i, f32x4_m{w[0][r], 0.f, 0.f, 0.f}, 1);
  }
};

struct PlaneMat {  // one matrix's planes in the workspace
  f16_t *x, *y, *a, *b;
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
  const float norm = (float)(sqrt(s) + (double)eps);
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
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        float x = 0.f;
        if (t + r < p.l) x = (tall ? tile[t - t0 + r][i - i0] : to_f(g[i * m.ldg + t + r])) / norm * kXs;
        f16_t v[2];
        split2(x, v);
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
  for (int i = 0; i < n; ++i) {
    const int s = sl[i][0], l = sl[i][1], ldx = up32(l), lda = up32(s);
    const long long xb = up256((long long)s * ldx * 4), ab = up256((long long)s * lda * 4);
    if (out) {
      f16_t* at = reinterpret_cast<f16_t*>(ws + w.bytes);
      out[i] = {at, at + xb / 2, at + xb, at + xb + ab / 2, s, l, lda, ldx};
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
void plane_iterate(const MatList& l, int n, char* ws, int steps, const float* co, float eps, int dt, const float* hyper,
                   hipStream_t st) {
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
               {p.a, nullptr, p.lda, p.s, ap, kAs / (kXs * kXs), 0.f}};
    jp.j[i] = {{p.a, p.lda, ap}, {p.a, p.lda, ap}, p.s, p.s, p.lda, 0, 0, 0, 0, nullptr,
               {p.b, p.a, p.lda, p.s, ap, co[2] / kAs, co[1]}};
    js.j[i] = {{p.b, p.lda, ap}, {p.x, p.ldx, xp}, p.s, p.l, p.s, 0, 0, 0, 0, nullptr,
               {p.y, p.x, xp, p.ldx, 0, 1.f / kAs, co[0], l.m[i].out, l.m[i].ldo, l.m[i].rows > l.m[i].cols,
                l.m[i].scale, hyper}};
  }
  const PlanePick pg = plane_pick<2, true>(gram, n), pp = plane_pick<2, true>(poly, n), ps = plane_pick<2, false>(step, n);
  for (int k = 0; k < steps; ++k) {
    plane_run<f16_t, 2, false, false, true>(jg, pg, part, st);
    plane_run<f16_t, 2, false, false, true>(jp, pp, part, st);
    if (k == steps - 1)
      for (int i = 0; i < n; ++i) js.j[i].e.mode = hyper ? 4 : 1 + dt;
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

// Whether iterates that start within |X| <= 1 stay where the planes hold them: |X| < 2^16 / kXs, |A| and |B|
// (largest entry <= largest singular value) < 2^16 / kAs
bool planes_hold(int steps, const float* co) {
  if (steps < 1) return false;
  double r = 1.0;
  for (int k = 0; k < steps; ++k) {
    if (r > 7.5 || std::fabs(co[1]) * r * r + std::fabs(co[2]) * r * r * r * r > 60.) return false;
    double next = 0;
    for (int q = 1; q <= 4096; ++q) {
      const double x = r * q / 4096, x2 = x * x;
      next = std::max(next, std::fabs(x * (co[0] + x2 * (co[1] + x2 * co[2]))));
    }
    r = next * 1.01;
  }
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
    if (r * c > 0) {
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
    if (m[i].rows < 0 || m[i].cols < 0) return "negative size";
    if ((long long)m[i].rows * m[i].cols == 0) continue;
    if (!m[i].g || !m[i].out) return "null matrix";
    if (m[i].ldg < m[i].cols || m[i].ldo < m[i].cols) return "row stride smaller than the row";
    const long long t = (std::max(m[i].rows, m[i].cols) + 63LL) / 64, u = (std::min(m[i].rows, m[i].cols) + 63LL) / 64;
    if (t * u > INT_MAX) return "matrix too large for one launch";
  }
  return nullptr;
}

Layout ortho_layout(const cgan3d_ortho_mat* m, int n) {
  Layout w = {};
  for (int i = 0; i < n; ++i) size_mat(w, m[i].rows, m[i].cols);
  place(w, n, 0, plane_bytes(n, [&](int i, long long& r, long long& c) { r = m[i].rows; c = m[i].cols; }));
  return w;
}

template <typename T>
void ortho_run(const cgan3d_ortho_mat* mats, int n, int dt, const Layout& w, char* ws, int steps, const float* co,
               float eps, hipStream_t st) {
  const bool planes = planes_hold(steps, co);
  MatList l;
  int at = 0;
  const auto flush = [&]() {
    if (!at) return;
    launch(norm_kernel<T>, dim3(kNormBlocks, at), dim3(256), 0, st, l);
    if (planes) {
      plane_iterate<T>(l, at, ws + w.x, steps, co, eps, dt, nullptr, st);
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
    if ((long long)q.rows * q.cols == 0) continue;
    l.m[at++] = {q.g, q.out, q.ldg, q.ldo, q.rows, q.cols, 1.f, reinterpret_cast<float*>(ws + w.x),
                 reinterpret_cast<double*>(ws + w.part) + (long long)i * kNormBlocks};
    if (at == (planes ? kJobs : 1)) flush();
  }
  flush();
}

const char* segs_check(const cgan3d_muon_seg* s, int n) {
  if (n < 0 || (n > 0 && !s)) return "null list";
  for (int i = 0; i < n; ++i) {
    if (s[i].offset < 0 || s[i].rows < 0 || s[i].cols < 0 || s[i].rows > INT_MAX) return "negative or too large size";
    if (s[i].rows > 0 && s[i].cols > INT_MAX) return "negative or too large size";
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
  place(w, nm, u, plane_bytes(n, [&](int i, long long& r, long long& c) { r = s[i].rows; c = s[i].cols; }));
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
  const Layout w = muon_layout(segs, n);
  CG_CHECK_ARG(ws_bytes >= w.total && (w.total == 0 || (ws && reinterpret_cast<uintptr_t>(ws) % 16 == 0)),
               "cgan3d_muon_step: workspace of %lld bytes (16-byte aligned) needed, got %lld", w.total,
               (long long)ws_bytes);
  hipStream_t st = (hipStream_t)stream;
  char* base = static_cast<char*>(ws);
  float* u = reinterpret_cast<float*>(base + w.u);
  double* part = reinterpret_cast<double*>(base + w.part);
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
    if (segs[i].rows > 0) {
      l.mat[at] = nm++;
      l.u[at] = uo / 4;
      uo += up256(total * 4);
    } else {
      l.mat[at] = -1;
    }
    if (!total) continue;
    l.s[at] = segs[i];
    if (++at == kList) flush();
  }
  flush();
  uo = 0;
  nm = 0;
  const bool planes = planes_hold(steps, coefficients);
  MatList q;
  int qn = 0;
  const auto run = [&]() {
    if (!qn) return;
    if (planes) {
      plane_iterate<float>(q, qn, base + w.x, steps, coefficients, eps, 0, hyper, st);
    } else {
      const unsigned blocks = (unsigned)std::min(((long long)q.m[0].rows * q.m[0].cols + 1023) / 1024, 4096LL);
      launch(scale_kernel<float>, dim3(blocks, 1), dim3(256), 0, st, q, eps);
      q.m[0].x = iterate(q.m[0], w, base, steps, coefficients, st);
      launch(muon_apply_kernel, dim3(blocks, 1), dim3(256), 0, st, q, (const float*)hyper);
    }
    qn = 0;
  };
  for (int i = 0; i < n; ++i) {
    if (segs[i].rows == 0) continue;
    const long long total = segs[i].rows * segs[i].cols;
    q.m[qn] = {u + uo / 4, param + segs[i].offset, segs[i].cols, segs[i].cols, (int)segs[i].rows, (int)segs[i].cols,
               segs[i].lr_scale, reinterpret_cast<float*>(base + w.x), part + (long long)nm * kNormBlocks};
    ++nm;
    uo += up256(total * 4);
    if (total && ++qn == (planes ? kJobs : 1)) run();
  }
  run();
  launch(muon_tick_kernel, dim3(1), dim3(1), 0, st, hyper);
  CG_LAUNCH_CHECK("cgan3d_muon_step");
  return CGAN3D_OK;
} catch (...) {
  set_error("cgan3d_muon_step: out of host memory");
  return CGAN3D_EHIP;
}
