// Matrix products C[I, J] = sum_t A(i, t) * B(j, t) of the linear block (linear.hip) and the
// Newton-Schulz iteration (muon.hip) on f32 instructions: the tile kernel that takes any size, stride and alignment.
//
// Either operand is "t-contiguous" (element (i, t) at i * ld + t: a row-major matrix whose columns are
// summed) or "t-strided" (element (i, t) at t * ld + i: its rows are summed), so the forward product,
// both gradients and the products of the iteration are one template.
#pragma once
#include <hip/hip_fp16.h>

#include "common.h"

namespace cg {

typedef _Float16 f16_t;
typedef __bf16 bf16_t;
typedef float f32x4_m __attribute__((ext_vector_type(4)));
typedef f16_t f16x4_m __attribute__((ext_vector_type(4)));
typedef bf16_t bf16x4_m __attribute__((ext_vector_type(4)));
typedef f16_t f16x8_m __attribute__((ext_vector_type(8)));
typedef bf16_t bf16x8_m __attribute__((ext_vector_type(8)));

template <typename T> struct MatT;
template <> struct MatT<float> { static constexpr int VEC = 4, PAD = 4; };
template <> struct MatT<f16_t> { static constexpr int VEC = 8, PAD = 8; };
template <> struct MatT<bf16_t> { static constexpr int VEC = 8, PAD = 8; };

template <typename T> __device__ __forceinline__ float to_f(T v) { return (float)v; }
// one rounding to nearest even on the way out of the 32-bit accumulators
template <typename T> __device__ __forceinline__ T from_f(float v) { return (T)v; }

// 16 x 16 x 32 (16-bit) or 8 x (16 x 16 x 4) (f32: element e of both 8-element fragments is one k of
// the instruction; the sum over t does not mind the order) on fragments of 8 t-values per lane:
// lane l holds row l % 16, t = (l / 16) * 8 .. + 7.  D: column (second operand's row) l % 16, rows
// (first operand's) (l / 16) * 4 + r.
__device__ __forceinline__ f32x4_m mfma_8(const bf16_t* a, const bf16_t* b, f32x4_m c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(*reinterpret_cast<const bf16x8_m*>(a),
                                                 *reinterpret_cast<const bf16x8_m*>(b), c, 0, 0, 0);
}
__device__ __forceinline__ f32x4_m mfma_8(const f16_t* a, const f16_t* b, f32x4_m c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_f16(*reinterpret_cast<const f16x8_m*>(a),
                                                *reinterpret_cast<const f16x8_m*>(b), c, 0, 0, 0);
}
__device__ __forceinline__ f32x4_m mfma_8(const float* a, const float* b, f32x4_m c) {
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const f32x4_m x = *reinterpret_cast<const f32x4_m*>(a + 4 * h), y = *reinterpret_cast<const f32x4_m*>(b + 4 * h);
#pragma unroll
    for (int e = 0; e < 4; ++e) c = __builtin_amdgcn_mfma_f32_16x16x4f32(x[e], y[e], c, 0, 0, 0);
  }
  return c;
}

// A vector at any address of whole elements: global memory takes accesses of up to 16 bytes unaligned, which then cost a
// second line now and then and not an access per value (4 x 7195 -> 253 f32 20 us, a value at a time 53; 1 x 4097 -> 4096
// bf16 8.5 and 26; 262144 x 15 -> 33 16 and 20).
template <typename V, typename T> __device__ __forceinline__ V load_v(const T* p) {
  V v;
  __builtin_memcpy(&v, p, sizeof(V));
  return v;
}
template <typename V, typename T> __device__ __forceinline__ void store_v(T* p, V v) { __builtin_memcpy(p, &v, sizeof(V)); }

// n of four neighbours (more than four: all)
template <typename T> __device__ __forceinline__ f32x4_m load4(const T* p, int n) {
  f32x4_m v = {0.f, 0.f, 0.f, 0.f};
  if (n >= 4) {
    typedef T v4 __attribute__((ext_vector_type(4)));
    const v4 x = load_v<v4>(p);
#pragma unroll
    for (int r = 0; r < 4; ++r) v[r] = to_f(x[r]);
  } else {
#pragma unroll
    for (int r = 0; r < 4; ++r)
      if (r < n) v[r] = to_f(p[r]);
  }
  return v;
}
template <typename T> __device__ __forceinline__ void store4(T* p, f32x4_m v, int n) {
  if (n >= 4) {
    typedef T v4 __attribute__((ext_vector_type(4)));
    v4 x;
#pragma unroll
    for (int r = 0; r < 4; ++r) x[r] = from_f<T>(v[r]);
    store_v(p, x);
  } else {
#pragma unroll
    for (int r = 0; r < 4; ++r)
      if (r < n) p[r] = from_f<T>(v[r]);
  }
}

// --- activations of the linear block (all in 32 bits) ---
// FAST: for 16-bit tensors, whose own rounding (2^-9 or 2^-12 of a value) hides the 2^-20 or so that these forms
// lose; the library's functions for f32 tensors.

// e^x by the hardware's 2^x
__device__ __forceinline__ float fast_exp(float x) { return __builtin_amdgcn_exp2f(x * 1.44269504088896341f); }
// Q(z) e^(z^2 / 2) for z >= 0, Q the normal distribution's upper tail: a polynomial in t = 1 / (1 + 0.3 z), fitted here
// by weighted least squares on Chebyshev points of t for an equal relative error over z < 14: 1.5e-7, 1e-6
// with its evaluation in f32.  Beyond, Q itself is below what the 16-bit types can tell from 0
__device__ __forceinline__ float normal_tail_scaled(float z) {
  const float t = __builtin_amdgcn_rcpf(1.f + 0.3f * z);
  float p = 0.035678383f;
  p = fmaf(p, t, -0.157217249f);
  p = fmaf(p, t, 0.206376284f);
  p = fmaf(p, t, -0.0537030324f);
  p = fmaf(p, t, 0.128571019f);
  p = fmaf(p, t, 0.0999109074f);
  p = fmaf(p, t, 0.120754331f);
  p = fmaf(p, t, 0.119629279f);
  return p * t;
}
// d/dz of z Phi(z) and z Phi(z) itself share the tail
__device__ __forceinline__ float fast_phi(float z, float* dens) {
  const float g = fast_exp(-0.5f * z * z), q = normal_tail_scaled(fabsf(z)) * g;
  *dens = g * 0.39894228040143268f;
  return z < 0.f ? q : 1.f - q;
}
__device__ __forceinline__ float fast_tanh(float z) {
  const float e = fast_exp(-2.f * fabsf(z));  // tanh |z| = (1 - e) / (1 + e); near 0 its own series
  const float b = (1.f - e) * __builtin_amdgcn_rcpf(1.f + e), z2 = z * z;
  const float s = fabsf(z) * (1.f + z2 * (-0.33333334f + z2 * (0.13333333f - z2 * 0.053968254f)));
  return copysignf(fabsf(z) < 0.125f ? s : b, z);
}

template <bool FAST> __device__ __forceinline__ float mat_act(float z, int act, float slope) {
  switch (act) {
    case CGAN3D_ACT_RELU: return z > 0.f ? z : (z == z ? 0.f : z);  // NaN stays NaN
    case CGAN3D_ACT_LRELU: return z > 0.f ? z : slope * z;
    case CGAN3D_ACT_TANH: return FAST ? fast_tanh(z) : tanhf(z);
    case CGAN3D_ACT_GELU: {
      if (!FAST) return 0.5f * z * (1.f + erff(z * 0.70710678118654752f));
      float d;
      return z * fast_phi(z, &d);
    }
    case CGAN3D_ACT_SILU: return FAST ? z * __builtin_amdgcn_rcpf(1.f + fast_exp(-z)) : z / (1.f + expf(-z));
  }
  return z;
}
// 16 values at once: one branch on the activation
template <typename T> __device__ __forceinline__ void mat_act16(float* v, int act, float slope) {
  constexpr bool FAST = sizeof(T) == 2;
#define CG_ACT16(A)                                     \
  case A:                                               \
    _Pragma("unroll") for (int q = 0; q < 16; ++q) v[q] = mat_act<FAST>(v[q], A, slope); \
    break;
  switch (act) {
    CG_ACT16(CGAN3D_ACT_RELU)
    CG_ACT16(CGAN3D_ACT_LRELU)
    CG_ACT16(CGAN3D_ACT_TANH)
    CG_ACT16(CGAN3D_ACT_GELU)
    CG_ACT16(CGAN3D_ACT_SILU)
  }
#undef CG_ACT16
}
// derivative at the pre-activation z.  The smooth ones are constant to the last bit of an f32 beyond
// |z| = 100, so z is clamped there: an infinite (or saturated, see mat_preact) z gives their limits,
// not inf * 0
template <bool FAST> __device__ __forceinline__ float mat_act_grad(float z, int act, float slope) {
  if (act == CGAN3D_ACT_RELU) return z > 0.f ? 1.f : 0.f;
  if (act == CGAN3D_ACT_LRELU) return z > 0.f ? 1.f : slope;
  if (act == CGAN3D_ACT_NONE) return 1.f;
  if (z == z) z = fminf(fmaxf(z, -100.f), 100.f);
  if (act == CGAN3D_ACT_TANH) {
    // 1 - tanh^2 = 4 e / (1 + e)^2, e = exp(-2 |z|): no cancellation where tanh is near 1
    const float e = FAST ? fast_exp(-2.f * fabsf(z)) : expf(-2.f * fabsf(z)), d = 1.f + e;
    return FAST ? 4.f * e * __builtin_amdgcn_rcpf(d * d) : 4.f * e / (d * d);
  }
  if (act == CGAN3D_ACT_GELU) {
    if (!FAST) return 0.5f * (1.f + erff(z * 0.70710678118654752f)) + z * expf(-0.5f * z * z) * 0.39894228040143268f;
    float d;
    const float phi = fast_phi(z, &d);
    return phi + z * d;
  }
  const float s = FAST ? __builtin_amdgcn_rcpf(1.f + fast_exp(-z)) : 1.f / (1.f + expf(-z));  // SiLU
  return s * (1.f + z * (1.f - s));
}

// The pre-activation kept for the backward pass: f32, but f16 for bf16 tensors.  Eleven bits of z leave act'(z) exact
// to well below bf16's own rounding of dz (eight would double that error) and save half the traffic; for f16
// tensors they would be as large as dz's rounding.  Values beyond f16's range saturate (act' is constant there),
// and a value that would round to zero keeps its sign in the smallest f16 (ReLU's derivative).
__device__ __forceinline__ void mat_preact(float* p, float z) { *p = z; }
__device__ __forceinline__ void mat_preact(f16_t* p, float z) {
  if (z == z) z = fminf(fmaxf(z, -65504.f), 65504.f);
  f16_t h = (f16_t)z;
  if (z != 0.f && h == (f16_t)0.f) h = z > 0.f ? (f16_t)5.9604645e-8f : (f16_t)-5.9604645e-8f;
  *p = h;
}
template <typename T> struct PreT { typedef float type; };
template <> struct PreT<bf16_t> { typedef f16_t type; };

// what happens to a product's element on its way out: v = alpha * acc + bias[j]; preact = v;
// v = act(v) + beta * residual[i, j]
struct MatEpi {
  const void* bias;
  const void* residual;
  long long ldr;
  void* preact;  // [I, J], PreT
  void* out;
  long long ldo;
  float alpha, beta;
  int act;
  float slope;
};

struct MatArgs {
  const void* a;
  const void* b;
  long long lda, ldb;
  long long I, J, K;
  long long tj;      // column tiles
  long long kchunk;  // t-values per split (whole K: one split)
  float* part;       // splits > 1: [split][I][J] partial sums
  MatEpi e;
};

template <typename T>
__device__ __forceinline__ void mat_store(const MatEpi& e, long long J, long long i, long long j, float acc) {
  float v = e.alpha * acc;
  if (e.bias) v += to_f(static_cast<const T*>(e.bias)[j]);
  if (e.preact) mat_preact(static_cast<typename PreT<T>::type*>(e.preact) + i * J + j, v);
  v = mat_act<sizeof(T) == 2>(v, e.act, e.slope);
  if (e.residual) v += e.beta * to_f(static_cast<const T*>(e.residual)[i * e.ldr + j]);
  static_cast<T*>(e.out)[i * e.ldo + j] = from_f<T>(v);
}

// One BM x BN tile, 4 waves as 2 x 2, BK t-values a step: global -> registers -> LDS (rows padded by
// 16 bytes), the next step's loads in flight under this step's products.  Bound by the f32 matrix instructions where it
// is used at all: 2048 x 1024 -> 4096 in 184 us, 4096 x 4096 -> 4096 in 1356, 93 and 101 TFLOP/s of 154 that a library
// product of 8192 reaches (what is larger goes to planes), and the iteration's fallback.
template <bool AT, bool BT, int BM, int BN>
__global__ __launch_bounds__(256) void mat_kernel(MatArgs p) {
  typedef float T;
  constexpr int BK = 32, V = MatT<T>::VEC, LD = BK + MatT<T>::PAD;
  constexpr int WM = BM / 2, WN = BN / 2, FM = WM / 16, FN = WN / 16;
  constexpr int NA = BM * BK / V / 256, NB = BN * BK / V / 256;  // 16-byte chunks per thread
  static_assert(NA >= 1 && NB >= 1 && BM * BK % (V * 256) == 0 && BN * BK % (V * 256) == 0, "whole chunks per thread");
  __shared__ __align__(16) T la[BM * LD];
  __shared__ __align__(16) T lb[BN * LD];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const long long ti = blockIdx.x / p.tj, tjj = blockIdx.x - ti * p.tj;
  const long long i0 = ti * BM, j0 = tjj * BN;
  const long long k0 = (long long)blockIdx.y * p.kchunk, k1 = std::min(p.K, k0 + p.kchunk);
  const int wi = (wave >> 1) * WM, wj = (wave & 1) * WN;
  f32x4_m acc[FN][FM] = {};
  typedef T vecT __attribute__((ext_vector_type(V)));
  vecT ra[NA], rb[NB];
  // one chunk of V values along the operand's contiguous axis: `inner` counts along it up to `ni`,
  // `outer` across it up to `no`; what is outside is zero
  auto load = [&](const T* base, long long ld, long long outer, long long no, long long inner, long long ni) {
    vecT v = {};
    if (outer < no && inner < ni) {
      const T* s = base + outer * ld + inner;
      if (inner + V <= ni) {
        v = load_v<vecT>(s);
      } else {
#pragma unroll
        for (int e = 0; e < V; ++e)
          if (inner + e < ni) v[e] = s[e];
      }
    }
    return v;
  };
  const T* A = static_cast<const T*>(p.a);
  const T* B = static_cast<const T*>(p.b);
  auto fetch = [&](long long k) {
#pragma unroll
    for (int c = 0; c < NA; ++c) {
      const int q = c * 256 + tid;
      if constexpr (AT) ra[c] = load(A, p.lda, k + q / (BM / V), k1, i0 + (q % (BM / V)) * V, p.I);
      else ra[c] = load(A, p.lda, i0 + q / (BK / V), p.I, k + (q % (BK / V)) * V, k1);
    }
#pragma unroll
    for (int c = 0; c < NB; ++c) {
      const int q = c * 256 + tid;
      if constexpr (BT) rb[c] = load(B, p.ldb, k + q / (BN / V), k1, j0 + (q % (BN / V)) * V, p.J);
      else rb[c] = load(B, p.ldb, j0 + q / (BK / V), p.J, k + (q % (BK / V)) * V, k1);
    }
  };
  auto put = [&]() {
#pragma unroll
    for (int c = 0; c < NA; ++c) {
      const int q = c * 256 + tid;
      if constexpr (AT) {
#pragma unroll
        for (int e = 0; e < V; ++e) la[((q % (BM / V)) * V + e) * LD + q / (BM / V)] = ra[c][e];
      } else {
        *reinterpret_cast<vecT*>(&la[q / (BK / V) * LD + (q % (BK / V)) * V]) = ra[c];
      }
    }
#pragma unroll
    for (int c = 0; c < NB; ++c) {
      const int q = c * 256 + tid;
      if constexpr (BT) {
#pragma unroll
        for (int e = 0; e < V; ++e) lb[((q % (BN / V)) * V + e) * LD + q / (BN / V)] = rb[c][e];
      } else {
        *reinterpret_cast<vecT*>(&lb[q / (BK / V) * LD + (q % (BK / V)) * V]) = rb[c];
      }
    }
  };
  if (k0 < k1) fetch(k0);
  for (long long k = k0; k < k1; k += BK) {
    __syncthreads();  // the previous step's reads are done
    put();
    __syncthreads();
    if (k + BK < k1) fetch(k + BK);
    const T* pa = &la[(wi + (lane & 15)) * LD + (lane >> 4) * 8];
    const T* pb = &lb[(wj + (lane & 15)) * LD + (lane >> 4) * 8];
#pragma unroll
    for (int n = 0; n < FN; ++n)
#pragma unroll
      for (int m = 0; m < FM; ++m) acc[n][m] = mfma_8(pb + n * 16 * LD, pa + m * 16 * LD, acc[n][m]);
  }
  // a lane holds four neighbouring columns j of one row i
#pragma unroll
  for (int m = 0; m < FM; ++m) {
    const long long i = i0 + wi + m * 16 + (lane & 15);
    if (i >= p.I) continue;
#pragma unroll
    for (int n = 0; n < FN; ++n) {
      const long long j = j0 + wj + n * 16 + (lane >> 4) * 4;
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        if (j + r >= p.J) break;
        if (p.part) p.part[((long long)blockIdx.y * p.I + i) * p.J + j + r] = acc[n][m][r];
        else mat_store<T>(p.e, p.J, i, j + r, acc[n][m][r]);
      }
    }
  }
}

// the splits' partial sums, added in their order (none: an empty sum), and the epilogue
template <typename T>
__global__ __launch_bounds__(256) void mat_join_kernel(MatArgs p, int splits) {
  const long long total = p.I * p.J;
  for (long long q = (long long)blockIdx.x * 256 + threadIdx.x; q < total; q += (long long)gridDim.x * 256) {
    float s = 0.f;
#pragma unroll 8
    for (int z = 0; z < splits; ++z) s += p.part[z * total + q];
    const long long i = q / p.J;
    mat_store<T>(p.e, p.J, i, q - i * p.J, s);
  }
}

// f32 product with its epilogue, splits and tiles chosen for the sizes (linear.hip); at / bt: that
// operand is t-strided.  Workspace: mat_f32_ws_bytes.
long long mat_f32_ws_bytes(long long I, long long J, long long K);
void mat_f32(bool at, bool bt, const MatArgs& p, void* ws, hipStream_t st);

}  // namespace cg
