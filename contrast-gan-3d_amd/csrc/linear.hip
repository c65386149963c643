// Linear block: y = act(x W^T + bias) + residual over rows of channels (a pointwise convolution over
// channels-last voxels), and its gradient.
//
//   z = x W^T + b            y = act(z) + r
//   dz = dy * act'(z)        dx = dz W        dW = dz^T x        db = sum over rows of dz        dr = dy
//
// The epilogue runs on the accumulators, so z, act(z) and the sum with r never pass through memory,
// apart from z itself where a backward pass will want it.
//
// Which kernel a product takes (mat_route):
//   rows <= 2, forward      gemv_kernel: a wave per pair of output columns streams the weight once
//   rows <= 16, forward     skinny_kernel: a wave per 16 columns, the weight straight into matrix instructions
//   k, n <= 64              rows_fwd_kernel, rows_bwd_kernel: every row's values are read and written once (16-bit ones
//                           with few rows: rows_fwd_takes, rows_bwd_takes)
//   16-bit tensors         plane_kernel (planes.h) on the tensors themselves; an operand whose rows are not
//                          whole aligned 16-byte chunks is copied once into rows that are
//   f32 tensors            plane_kernel on three bf16 planes where that is expected to be faster (f32_planes), else
//                          mat_kernel (mat.h: f32 instructions, any layout)
#include <climits>

#include "planes.h"

namespace cg {
namespace {

constexpr int kTile = 64;

int dt_bytes(int dt) { return dt == CGAN3D_DT_F32 ? 4 : 2; }
int pre_bytes(int dt) { return dt == CGAN3D_DT_BF16 ? 2 : 4; }

// Splits of mat_kernel's summed axis: as many as fill the card twice, each at least 256 values long.
int mat_splits(long long I, long long J, long long K) {
  const long long tiles = std::max(1LL, ((I + kTile - 1) / kTile) * ((J + kTile - 1) / kTile));
  const long long want = 2LL * cu_count() / tiles, most = K / 256;
  return (int)std::max(1LL, std::min({want, most, 1024LL}));
}
long long mat_ws_bytes(long long I, long long J, long long K) {
  const int s = mat_splits(I, J, K);
  return s > 1 ? (long long)s * I * J * 4 : 0;
}

template <bool AT, bool BT>
void mat_run(MatArgs p, void* ws, hipStream_t st) {
  if (p.I == 0 || p.J == 0) return;
  int splits = mat_splits(p.I, p.J, p.K);
  const long long steps = (p.K + 31) / 32;
  p.kchunk = std::max(1LL, (steps + splits - 1) / splits) * 32;
  splits = (int)std::max(1LL, (p.K + p.kchunk - 1) / p.kchunk);
  p.part = splits > 1 ? static_cast<float*>(ws) : nullptr;
  const long long ti = (p.I + kTile - 1) / kTile;
  p.tj = (p.J + kTile - 1) / kTile;
  launch(mat_kernel<AT, BT, kTile, kTile>, dim3((unsigned)(ti * p.tj), splits), dim3(256), 0, st, p);
  if (splits > 1) {
    const long long blocks = std::min((p.I * p.J + 255) / 256, 8192LL);
    launch(mat_join_kernel<float>, dim3((unsigned)blocks), dim3(256), 0, st, p, splits);
  }
}
// an empty sum: the epilogue of zeros
void mat_zero(int dt, const MatArgs& p, hipStream_t st) {
  const dim3 grid((unsigned)std::min((p.I * p.J + 255) / 256, 8192LL));
  if (dt == CGAN3D_DT_F32) launch(mat_join_kernel<float>, grid, dim3(256), 0, st, p, 0);
  else if (dt == CGAN3D_DT_BF16) launch(mat_join_kernel<bf16_t>, grid, dim3(256), 0, st, p, 0);
  else launch(mat_join_kernel<f16_t>, grid, dim3(256), 0, st, p, 0);
}

// --- products on planes ---

// Epilogue of a plane product.  NANFIX (f32 on three planes): an infinity times an empty lower plane
// is NaN, and a first plane that was rounded up can overflow where the value's own product does not, so a sum that is
// not finite is computed again value by value, which leaves what f32 gives (2048 x 1024 -> 4096: 122 us, with a row that
// is not finite 477, with nothing but infinite sums 8600).
template <typename T, bool NANFIX> struct LinEpi {
  static constexpr bool STAGED = true;
  MatEpi e;
  long long J;
  struct Values {  // NANFIX: an operand's planes; element (i, t) at i si + t st
    const bf16_t* p;
    long long plane, si, st;
    __device__ __forceinline__ float at(long long i, long long t) const {
      const bf16_t* q = p + i * si + t * st;
      return ((float)q[0] + (float)q[plane]) + (float)q[2 * plane];
    }
    // t .. t + 7, t a multiple of 8: whole chunks of a row, or eight rows
    __device__ __forceinline__ void eight(long long i, long long t, float (&o)[8]) const {
      if (st == 1) {
        const bf16_t* q = p + i * si + t;
        const bf16x8_m h = load_v<bf16x8_m>(q), m = load_v<bf16x8_m>(q + plane), l = load_v<bf16x8_m>(q + 2 * plane);
#pragma unroll
        for (int e = 0; e < 8; ++e) o[e] = ((float)h[e] + (float)m[e]) + (float)l[e];
      } else {
#pragma unroll
        for (int e = 0; e < 8; ++e) o[e] = at(i, t + e);
      }
    }
  };
  Values a, b;
  long long K;
  __device__ __noinline__ float again(int i, int j) const {
    float s = 0.f;
    long long t = 0;
    for (; t + 8 <= K && s == s; t += 8) {  // eight loads in flight; NaN stays NaN
      float x[8], y[8];
      a.eight(i, t, x);
      b.eight(j, t, y);
#pragma unroll
      for (int q = 0; q < 8; ++q) s = fmaf(x[q], y[q], s);
    }
    for (; t < K && s == s; ++t) s = fmaf(a.at(i, t), b.at(j, t), s);
    return s;
  }
  // V: all four columns are there
  template <int STEP, bool V> __device__ __forceinline__ void put4_as(int i, int j, f32x4_m* v, int I, int jn) const {
    typedef typename PreT<T>::type preT;
    typedef T v4 __attribute__((ext_vector_type(4)));
    // as they are until they are needed; columns that are not there: the last one again, without a branch (a
    // load under a branch is waited for by itself)
    const auto fetch = [&](const T* row) {
      v4 x;
      if (V) return load_v<v4>(row + j);
#pragma unroll
      for (int r = 0; r < 4; ++r) x[r] = row[j + min(r, jn - 1)];
      return x;
    };
    v4 res[4], bias;
    if (e.bias) bias = fetch(static_cast<const T*>(e.bias));
    if (e.residual) {
#pragma unroll
      for (int u = 0; u < 4; ++u) res[u] = fetch(static_cast<const T*>(e.residual) + min(i + u * STEP, I - 1) * e.ldr);
    }
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      v[u] *= e.alpha;
      if (e.bias) {
#pragma unroll
        for (int r = 0; r < 4; ++r) v[u][r] += to_f(bias[r]);
      }
      if (e.preact && i + u * STEP < I) {
        typedef preT p4 __attribute__((ext_vector_type(4)));
        preT* o = static_cast<preT*>(e.preact) + (i + u * STEP) * J + j;
        p4 p;
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          preT q;
          mat_preact(&q, v[u][r]);
          p[r] = q;
        }
        if (V) store_v(o, p);
        else
#pragma unroll
          for (int r = 0; r < 4; ++r)
            if (r < jn) o[r] = p[r];
      }
    }
    mat_act16<T>(reinterpret_cast<float*>(v), e.act, e.slope);
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      if (i + u * STEP >= I) continue;
      if (e.residual) {
#pragma unroll
        for (int r = 0; r < 4; ++r) v[u][r] += e.beta * to_f(res[u][r]);
      }
      store4(static_cast<T*>(e.out) + (i + u * STEP) * e.ldo + j, v[u], jn);
    }
  }
  // four columns from j of rows i, i + STEP, .. + 3 STEP: every load before the first store, so that they are in
  // flight together
  template <int STEP>
  __device__ __forceinline__ void put4(int i, int j, f32x4_m* v, int I, int jn, int) const {
    if constexpr (NANFIX) {
#pragma unroll
      for (int u = 0; u < 4; ++u)
#pragma unroll
        for (int r = 0; r < 4; ++r)
          if (i + u * STEP < I && r < jn && !(fabsf(v[u][r]) < __builtin_inff())) v[u][r] = again(i + u * STEP, j + r);
    }
    if (jn >= 4) put4_as<STEP, true>(i, j, v, I, 4);
    else put4_as<STEP, false>(i, j, v, I, jn);
  }
  __device__ __forceinline__ int begin() const { return 0; }
  __device__ __forceinline__ bool turned() const { return false; }
  __device__ __forceinline__ void put_turned(int, int, f32x4_m, int) const {}
  // the joined sums, a row at a time
  __device__ __forceinline__ void put(int i, int j, f32x4_m v, int jn, bool, int) const {
    f32x4_m w[4] = {v};
    put4<1>(i, j, w, i + 1, jn, 0);
  }
};

// An operand as planes, both of a product in one launch (bound by memory, or by the launch: 777 x 1001 and 515 x 1001 of
// f16 5.9 us).  Copied (16-bit) or split (f32) into rows of whole chunks, padding zeroed
struct Pack {
  const void* src;
  long long ld, rows;
  int cols, ldp;
  void* dst;
  long long first;  // chunk number of the launch at which this operand starts
};
struct Packs {
  Pack p[2];
  long long chunks;
};
// Row length of planes: whole 16-byte chunks, and whole 128-byte lines where that adds little: the products fetch 64 bytes
// of each row at a time, which else lie in two lines (bf16 97852 x 520 -> 1024, us by row length: 520 196, 544 186, 576
// 165; 8192 x 1000 -> 1024: 1000 33.6, 1008 31.4, 1024 28.1).
long long row_pad(long long cols) { return cols >= 256 ? (cols + 63) / 64 * 64 : (cols + 7) / 8 * 8; }
long long up256(long long v) { return (v + 255) / 256 * 256; }

template <typename T>
__global__ __launch_bounds__(256) void pack_kernel(Packs ps) {
  for (long long q = (long long)blockIdx.x * 256 + threadIdx.x; q < ps.chunks; q += gridDim.x * 256LL) {
    const Pack& p = ps.p[q >= ps.p[1].first];
    const long long u = q - p.first;
    const int nc = p.ldp / 8;
    const long long row = u / nc;
    const int c = (int)(u - row * nc) * 8;
    const T* s = static_cast<const T*>(p.src) + row * p.ld + c;
    __align__(16) T v[8];
    if (c + 8 <= p.cols) {
      __builtin_memcpy(v, s, sizeof(v));
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] = c + e < p.cols ? s[e] : from_f<T>(0.f);
    }
    if constexpr (sizeof(T) == 4) {
      const long long plane = p.rows * p.ldp, o = row * p.ldp + c;
      bf16x8_m h, m, l;
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        bf16_t t[3];
        split3(v[e], t);
        h[e] = t[0];
        m[e] = t[1];
        l[e] = t[2];
      }
      bf16_t* d = static_cast<bf16_t*>(p.dst) + o;
      *reinterpret_cast<bf16x8_m*>(d) = h;
      *reinterpret_cast<bf16x8_m*>(d + plane) = m;
      *reinterpret_cast<bf16x8_m*>(d + 2 * plane) = l;
    } else {
      typedef T v8 __attribute__((ext_vector_type(8)));
      *reinterpret_cast<v8*>(static_cast<T*>(p.dst) + row * p.ldp + c) = *reinterpret_cast<v8*>(v);
    }
  }
}

bool chunked(const void* p, long long ld, long long cols) {
  return reinterpret_cast<uintptr_t>(p) % 16 == 0 && ld % 8 == 0 && cols % 8 == 0;
}

// One operand of a product: [rows, cols] with row stride ld; `strided`: its rows are summed over.
struct Operand {
  const void* p;
  long long ld, rows;
  int cols;
  bool strided;
  bool planes;  // p already holds planes (dz), rows of ld values
};

enum Route { ROUTE_MAT, ROUTE_PLANES };

// What an f32 product is expected to take.  On f32 instructions: the rounds of tiles that the fullest CU gets, at 100
// TFLOP/s of the card, a tenth more where an operand is turned on its way to LDS, and each round's start; the output;
// the launch, and the join of split sums.  On planes: plane_pick's own estimate, the splitting, the output and three launches.
// Measured, us, f32 instructions / planes, what is taken in brackets.  Forward: rows x k -> n 2048 x 512 -> 1024 29.6 / 40.5
// (f), 1500 x 1000 -> 1203 51 / 56 (f), 8191 x 65 -> 4099 109 / 133 (f), 2048 x 1024 -> 2048 96 / 68 (p), 2500 x 777 -> 1111
// 58 / 56 (f); dx and dw: 1300 x 700 -> 900 37 / 33 (p) and 38 / 46 (f), 6001 x 203 -> 2999 205 / 105 (p) and 273 / 104 (p),
// 4096 x 256 -> 1024 41 / 35 (f) and 40 / 39 (f).  Over 30 sizes the slower form costs 0.6 % on average, 16 % once.
double mat_seconds(const Operand& a, const Operand& b, long long I, long long J, long long K) {
  const int splits = mat_splits(I, J, K), cus = cu_count();
  const double tiles = (double)((I + kTile - 1) / kTile) * ((J + kTile - 1) / kTile) * splits;
  const double len = std::ceil(std::ceil(K / 32.) / splits) * 32;
  const double tile = 2. * kTile * kTile * len / (100e12 / cus) * (b.strided ? 1.1 : 1.) + (a.strided ? 1.5e-6 : b.strided ? 8e-7 : 0);
  return std::ceil(tiles / cus) * tile + 4. * I * J / 2.7e12 + 4e-6 + (splits > 1 ? 9e-6 : 0);
}
double planes_seconds(const Operand& a, const Operand& b, long long I, long long J, long long K) {
  const PlaneShape s = {(int)I, (int)J, (int)K};
  double values = 0;
  for (const Operand* o : {&a, &b})
    if (!o->planes) values += (double)o->rows * row_pad(o->cols);
  return 0.7 * plane_pick<3, false>(&s, 1).seconds + values * 10 / 8e12 + 4. * I * J / 1.95e12 + 15e-6;
}
bool f32_planes(const Operand& a, const Operand& b, long long I, long long J, long long K) {
  const double m = mat_seconds(a, b, I, J, K);  // planes take 15 us at least: no estimate needed below that
  return m > 15e-6 && m > planes_seconds(a, b, I, J, K);
}
Route mat_route(int dt, const Operand& a, const Operand& b, long long I, long long J, long long K) {
  return dt != CGAN3D_DT_F32 || a.planes || f32_planes(a, b, I, J, K) ? ROUTE_PLANES : ROUTE_MAT;
}

long long operand_bytes(int dt, const Operand& o) {
  if (o.planes) return 0;
  if (dt == CGAN3D_DT_F32) return up256(o.rows * row_pad(o.cols) * 6);
  return chunked(o.p, o.ld, o.cols) ? 0 : up256(o.rows * row_pad(o.cols) * 2);
}
PlanePick pick_for(int dt, long long I, long long J, long long K) {
  const PlaneShape s = {(int)I, (int)J, (int)K};
  return dt == CGAN3D_DT_F32 ? plane_pick<3, false>(&s, 1) : plane_pick<1, false>(&s, 1);
}
// Whether the product's launches are ones that HIP takes: fewer than 2^32 threads along x, sides that the kernels count in
// 32 bits
template <int P> long long plane_threads(const PlanePick& p, const PlaneShape& s) {
  using C = PlaneCfg<P, false>;
  return plane_tiles(s, C::BM[p.cfg], C::BN[p.cfg], false) * std::max(1, (s.K + p.kchunk - 1) / p.kchunk) * C::WI[p.cfg] *
         C::WJ[p.cfg] * 64;
}
bool launchable(int dt, long long I, long long J, long long K) {
  const long long side = 1LL << 30, tiles = (I + kTile - 1) / kTile * ((J + kTile - 1) / kTile);
  if (I == 0 || J == 0) return true;
  if (I > side || J > side || K > side) return false;
  if (tiles < 1 << 22) return true;  // of the smallest tile; no block has more than 512 threads, splits come with few tiles
  const PlaneShape s = {(int)I, (int)J, (int)K};
  const PlanePick p = pick_for(dt, I, J, K);
  if (dt != CGAN3D_DT_F32) return plane_threads<1>(p, s) < 1LL << 32;
  return plane_threads<3>(p, s) < 1LL << 32 && tiles * 256 < 1LL << 32;
}
// workspace of one product: both operands' planes, then partial sums
long long product_bytes(int dt, const Operand& a, const Operand& b, long long I, long long J, long long K) {
  if (I == 0 || J == 0 || K == 0) return 0;
  if (mat_route(dt, a, b, I, J, K) == ROUTE_MAT) return mat_ws_bytes(I, J, K);
  return operand_bytes(dt, a) + operand_bytes(dt, b) + pick_for(dt, I, J, K).part_floats * 4;
}

template <typename T, typename PT, int P>
void planes_run(int dt, Operand a, Operand b, const MatArgs& m, void* ws, hipStream_t st) {
  char* at = static_cast<char*>(ws);
  Packs ps = {};
  const Operand a0 = a, b0 = b;
  int np = 0;
  Operand* os[2] = {&a, &b};
  for (Operand* o : os) {
    const long long bytes = operand_bytes(dt, *o);
    if (!bytes) continue;
    const int ldp = (int)row_pad(o->cols);
    ps.p[np++] = {o->p, o->ld, o->rows, o->cols, ldp, at, ps.chunks};
    ps.chunks += o->rows * (ldp / 8);
    o->p = at;
    o->ld = ldp;
    at += bytes;
  }
  if (np == 1) ps.p[1].first = LLONG_MAX;
  if (ps.chunks)
    launch(pack_kernel<T>, dim3((unsigned)std::min((ps.chunks + 255) / 256, 16384LL)), dim3(256), 0, st, ps);
  PlaneJobs<LinEpi<T, P == 3>, 1> jobs;
  jobs.n = 1;
  auto& j = jobs.j[0];
  j.a = {a.p, a.ld, a.rows * a.ld};
  j.b = {b.p, b.ld, b.rows * b.ld};
  j.I = (int)m.I;
  j.J = (int)m.J;
  j.K = (int)m.K;
  j.e.e = m.e;
  j.e.J = m.J;
  if constexpr (P == 3) {
    j.e.a = {static_cast<const bf16_t*>(a.p), a.rows * a.ld, a.strided ? 1 : a.ld, a.strided ? a.ld : 1};
    j.e.b = {static_cast<const bf16_t*>(b.p), b.rows * b.ld, b.strided ? 1 : b.ld, b.strided ? b.ld : 1};
    j.e.K = m.K;
  }
  const PlanePick pick = pick_for(dt, m.I, m.J, m.K);
  if (a0.strided) plane_run<PT, P, true, true, false>(jobs, pick, reinterpret_cast<float*>(at), st);
  else if (b0.strided) plane_run<PT, P, false, true, false>(jobs, pick, reinterpret_cast<float*>(at), st);
  else plane_run<PT, P, false, false, false>(jobs, pick, reinterpret_cast<float*>(at), st);
}

// C = A B^T with m's epilogue; m.a / m.b: the operands as the tensors they are
void product(int dt, const Operand& a, const Operand& b, const MatArgs& m, void* ws, hipStream_t st) {
  if (m.I == 0 || m.J == 0) return;
  if (m.K == 0) {
    mat_zero(dt, m, st);
  } else if (mat_route(dt, a, b, m.I, m.J, m.K) == ROUTE_MAT) {
    mat_f32(a.strided, b.strided, m, ws, st);
  } else if (dt == CGAN3D_DT_F32) {
    planes_run<float, bf16_t, 3>(dt, a, b, m, ws, st);
  } else if (dt == CGAN3D_DT_BF16) {
    planes_run<bf16_t, bf16_t, 1>(dt, a, b, m, ws, st);
  } else {
    planes_run<f16_t, f16_t, 1>(dt, a, b, m, ws, st);
  }
}

// A grid along x and, where that would be 2^32 threads or more (HIP refuses it), y too.  Blocks past the last find nothing
// to do.
dim3 long_grid(long long blocks, int threads) {
  const long long x = std::min(blocks, (1LL << 31) / threads);
  return dim3((unsigned)x, (unsigned)((blocks + x - 1) / x));
}
__device__ __forceinline__ int long_block() { return blockIdx.x + gridDim.x * blockIdx.y; }

// --- one or two rows: the weight is read once, 16 bytes a lane, and nothing else matters ---
// Bound by memory.  A wave takes R = 2 columns of y, so that a load of x serves two of the weight; KW waves of the block
// share the summed axis: 4, unless a wave would then get less than one load a column and the columns alone fill
// the card.  Measured, us, KW = 1 / 4, two rows: bf16 4096 -> 4096 10.8 / 8.5, 2048 -> 16384 15.7 / 13.2, 1024 -> 8192
// 6.1 / 6.9, 512 -> 16384 6.2 / 10.9; f32 1024 -> 8192 10.1 / 8.4.  One row, weights from memory: bf16 4096 -> 4096 8.0 us
// (4.2 TB/s), f32 13.2 (5.1 TB/s).  From three rows on the products and conversions in the vector unit take as
// long as the loads, and skinny_kernel is faster (four rows, bf16 4096 -> 4096: 12.0 here, 9.0 there).
constexpr int kGemvRows = 2;
template <typename T, int M, int KW>
__global__ __launch_bounds__(256) void gemv_kernel(const T* __restrict__ x, long long ldx, const T* __restrict__ w,
                                                   long long ldw, int n, int k, MatEpi e) {
  constexpr int V = MatT<T>::VEC, R = 2;
  typedef T vecT __attribute__((ext_vector_type(V)));
  __shared__ float red[4][M * R];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, part = wave % KW;
  const int j0 = (long_block() * (4 / KW) + wave / KW) * R;
  float acc[M][R] = {};
  if (j0 < n) {
    const T* wr[R];
#pragma unroll
    for (int r = 0; r < R; ++r) wr[r] = w + std::min(j0 + r, n - 1) * ldw;
    int t = (part * 64 + lane) * V;
#pragma unroll 4
    for (; t + V <= k; t += KW * 64 * V) {
      vecT xv[M], wv[R];
#pragma unroll
      for (int r = 0; r < R; ++r) wv[r] = load_v<vecT>(wr[r] + t);
#pragma unroll
      for (int m = 0; m < M; ++m) xv[m] = load_v<vecT>(x + m * ldx + t);
#pragma unroll
      for (int m = 0; m < M; ++m)
#pragma unroll
        for (int r = 0; r < R; ++r)
#pragma unroll
          for (int q = 0; q < V; ++q) acc[m][r] = fmaf(to_f(xv[m][q]), to_f(wv[r][q]), acc[m][r]);
    }
    // the last values
    for (; t < k; t += KW * 64 * V)
      for (int q = 0; q < V && t + q < k; ++q)
#pragma unroll
        for (int m = 0; m < M; ++m)
#pragma unroll
          for (int r = 0; r < R; ++r) acc[m][r] = fmaf(to_f(x[m * ldx + t + q]), to_f(wr[r][t + q]), acc[m][r]);
  }
#pragma unroll
  for (int m = 0; m < M; ++m)
#pragma unroll
    for (int r = 0; r < R; ++r) acc[m][r] = wave_sum(acc[m][r]);
  if constexpr (KW > 1) {
    if (lane == 0)
#pragma unroll
      for (int q = 0; q < M * R; ++q) red[wave][q] = acc[q / R][q % R];
    __syncthreads();
    if (wave == 0 && lane < M * R && j0 + lane % R < n)
      mat_store<T>(e, n, lane / R, j0 + lane % R, (red[0][lane] + red[1][lane]) + (red[2][lane] + red[3][lane]));
  } else {
#pragma unroll
    for (int q = 0; q < M * R; ++q)
      if (lane == q && j0 + q % R < n) mat_store<T>(e, n, q / R, j0 + q % R, acc[q / R][q % R]);
  }
}

template <typename T, int M> void gemv_run_m(const MatArgs& p, hipStream_t st) {
  const T* x = static_cast<const T*>(p.a);
  const T* w = static_cast<const T*>(p.b);
  const int V = MatT<T>::VEC, n = (int)p.J, k = (int)p.K;
  if (k < 4 * 64 * V && n / 2 >= 8 * cu_count())
    launch(gemv_kernel<T, M, 1>, long_grid((n + 7) / 8, 256), dim3(256), 0, st, x, p.lda, w, p.ldb, n, k, p.e);
  else
    launch(gemv_kernel<T, M, 4>, long_grid((n + 1) / 2, 256), dim3(256), 0, st, x, p.lda, w, p.ldb, n, k, p.e);
}
template <typename T> void gemv_run(const MatArgs& p, hipStream_t st) {
  if (p.I == 1) gemv_run_m<T, 1>(p, st);
  else gemv_run_m<T, 2>(p, st);
}

// n of eight neighbours (more: all), zeros for the others
template <typename T> __device__ __forceinline__ void load8(const T* p, int n, T (&v)[8]) {
  if (n >= 8) {
    __builtin_memcpy(v, p, sizeof(v));
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = e < n ? p[e] : from_f<T>(0.f);
  }
}

// --- up to 16 rows: a wave per 16 columns, weight and rows straight from memory into fragments ---
// Bound by memory (and, with 16 rows of many columns, by the rows' own way through L2: each block reads all of them).
// No LDS but for the join: a value of the weight is used once.  The KW waves of a block share the summed axis, U steps
// of 32 values each in flight; 16 waves where each has U steps to do, else 4.  Measured, us, KW = 4 / 16, 8 rows: bf16
// 4096 -> 4096 11.1 / 9.5 (3.5 TB/s), 2048 -> 4096 6.3 / 8.4; f32 4096 -> 4096 18.9 / 16.7, 2048 -> 4096 11.4 / 9.7,
// 1024 -> 8192 10.1 / 15.7.  With more than 32 columns a CU, four waves from ten rows on (f32 16 x 8192 -> 16384 126 / 133,
// 10 x 110 / 118, 8 x 8192 -> 32768 231 / 219, 3 x 230 / 204).  As products of tiles (planes, mat_kernel) the first five
// take 12.9, 9.8, 28, 17.5 and 18.5.
// 16-bit weights with more columns than 32 a CU are the planes' (16 rows, 4096 -> 16384: 40 here, 33 there; 2048 ->
// 16384: 22 and 18), f32 ones are not (68 and 96).
constexpr int kSkinnyRows = 16;
template <typename T> constexpr int kSkinnySteps = sizeof(T) == 2 ? 8 : 4;
template <typename T, int KW>
__global__ __launch_bounds__(KW * 64) void skinny_kernel(const T* __restrict__ x, long long ldx, const T* __restrict__ w,
                                                         long long ldw, int rows, int n, int k, MatEpi e) {
  constexpr int U = kSkinnySteps<T>;
  __shared__ f32x4_m red[KW][64];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), row = lane & 15, g = lane >> 4;
  const int j0 = long_block() * 16;
  // rows that are not there: the last one again
  const T* wr = w + (long long)min(j0 + row, n - 1) * ldw + g * 8;
  const T* xr = x + (long long)min(row, rows - 1) * ldx + g * 8;
  f32x4_m acc = {};
  const int full = k / 32;
  for (int s0 = wave; s0 < full; s0 += KW * U) {
    __align__(16) T fw[U][8], fx[U][8];
#pragma unroll
    for (int u = 0; u < U; ++u) {  // behind the last step: that one again, as zeros
      const int s = min(s0 + u * KW, full - 1) * 32;
      load8(wr + s, 8, fw[u]);
      load8(xr + s, 8, fx[u]);
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (u > 0 && s0 + u * KW >= full)
#pragma unroll
        for (int q = 0; q < 8; ++q) fw[u][q] = fx[u][q] = from_f<T>(0.f);
      acc = mfma_8(fw[u], fx[u], acc);
    }
  }
  if (wave == 0 && full * 32 < k) {
    __align__(16) T fw[8], fx[8];
    load8(wr + full * 32, k - full * 32 - g * 8, fw);
    load8(xr + full * 32, k - full * 32 - g * 8, fx);
    acc = mfma_8(fw, fx, acc);
  }
  red[wave][lane] = acc;
  __syncthreads();
  const int i = threadIdx.x / 16, j = threadIdx.x % 16;
  if (threadIdx.x < 256 && i < rows && j0 + j < n) {
    float v = 0.f;
#pragma unroll
    for (int z = 0; z < KW; ++z) v += red[z][j / 4 * 16 + i][j % 4];
    mat_store<T>(e, n, i, j0 + j, v);
  }
}
template <typename T> void skinny_run(const MatArgs& p, hipStream_t st) {
  const T* x = static_cast<const T*>(p.a);
  const T* w = static_cast<const T*>(p.b);
  const int n = (int)p.J, k = (int)p.K;
  const int blocks = (n + 15) / 16;
  if (k >= 16 * 32 * kSkinnySteps<T> && (p.I < 10 || n <= 32 * cu_count()))
    launch(skinny_kernel<T, 16>, long_grid(blocks, 1024), dim3(1024), 0, st, x, p.lda, w, p.ldb, (int)p.I, n, k, p.e);
  else launch(skinny_kernel<T, 4>, long_grid(blocks, 256), dim3(256), 0, st, x, p.lda, w, p.ldb, (int)p.I, n, k, p.e);
}

// --- few channels (k, n <= 64): every row's values are read and written once ---
// Forward: a wave takes 16 rows at a time, x straight from memory into fragments, the whole weight in registers; no
// LDS, no barrier.  Bound by memory where there are many rows (1048576 x 64 -> 64: f32 150 us, 3.6 TB/s, bf16 57 us,
// 4.7 TB/s; the products' own kernels 198 and 77), by the launch and one trip for the weight and one for the rows where
// there are few (4096 x 64 -> 64: f32 6.7 us against 7.3, bf16 4.8 against 4.0, 16 -> 16 3.6 against 3.9).
template <typename T, int NT, int KS>
__global__ __launch_bounds__(256) void rows_fwd_kernel(const T* __restrict__ x, long long ldx, const T* __restrict__ w,
                                                       long long ldw, long long rows, int n, int k, MatEpi e) {
  typedef T v4 __attribute__((ext_vector_type(4)));
  typedef typename PreT<T>::type preT;
  typedef preT p4 __attribute__((ext_vector_type(4)));
  const int lane = threadIdx.x & 63, row = lane & 15, g = lane >> 4;
  __align__(16) T fw[NT][KS][8];
#pragma unroll
  for (int t = 0; t < NT; ++t)
#pragma unroll
    for (int s = 0; s < KS; ++s) {
      const int j = t * 16 + row, c = s * 32 + g * 8;
      load8(w + (long long)min(j, n - 1) * ldw + c, j < n ? k - c : 0, fw[t][s]);
    }
  v4 bias[NT] = {};
  if (e.bias)
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
      for (int r = 0; r < 4; ++r)
        if (t * 16 + g * 4 + r < n) bias[t][r] = static_cast<const T*>(e.bias)[t * 16 + g * 4 + r];
  const long long groups = (rows + 15) / 16, step = (long long)gridDim.x * 4;
  for (long long q = (long long)blockIdx.x * 4 + (threadIdx.x >> 6); q < groups; q += step) {
    const long long i = q * 16 + row;
    const bool in = i < rows;
    __align__(16) T fx[KS][8];
    v4 res[NT];
#pragma unroll
    for (int s = 0; s < KS; ++s) load8(x + i * ldx + s * 32 + g * 8, in ? k - (s * 32 + g * 8) : 0, fx[s]);
    if (e.residual && in)
#pragma unroll
      for (int t = 0; t < NT; ++t)
        if (t * 16 + g * 4 + 4 <= n) res[t] = load_v<v4>(static_cast<const T*>(e.residual) + i * e.ldr + t * 16 + g * 4);
    f32x4_m acc[NT] = {};
#pragma unroll
    for (int s = 0; s < KS; ++s)
#pragma unroll
      for (int t = 0; t < NT; ++t) acc[t] = mfma_8(fw[t][s], fx[s], acc[t]);
    if (!in) continue;
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      const int j = t * 16 + g * 4;
      if (j >= n) continue;
      f32x4_m v = acc[t];
      if (j + 4 > n) {
#pragma unroll
        for (int r = 0; r < 4; ++r)
          if (j + r < n) mat_store<T>(e, n, i, j + r, v[r]);
        continue;
      }
      if (e.bias)
#pragma unroll
        for (int r = 0; r < 4; ++r) v[r] += to_f(bias[t][r]);
      if (e.preact) {
        p4 p;
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          preT z;
          mat_preact(&z, v[r]);
          p[r] = z;
        }
        store_v(static_cast<preT*>(e.preact) + i * n + j, p);
      }
      v4 o;
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        v[r] = mat_act<sizeof(T) == 2>(v[r], e.act, e.slope);
        o[r] = from_f<T>(e.residual ? v[r] + to_f(res[t][r]) : v[r]);
      }
      store_v(static_cast<T*>(e.out) + i * e.ldo + j, o);
    }
  }
}

// Backward: one pass over dy, z and x writes dx and keeps dW and db in registers; a block takes tiles of 64 rows in
// turn and leaves one partial sum of each.  dz is used as its own type would hold it, for db before that.  dz and x go
// through LDS in both orders, since one product sums over columns and the other over rows: that, not memory, bounds
// the 16-bit form (1048576 x 64 -> 64 with SiLU: f32 344 us, 3.1 TB/s, bf16 235 us, 2.3 TB/s).
constexpr int kRowsBlocks = 512;
template <typename T, int NT, int KT>
__global__ __launch_bounds__(256) void rows_bwd_kernel(const T* __restrict__ dy, long long lddy,
                                                       const typename PreT<T>::type* __restrict__ pre,
                                                       const T* __restrict__ x, long long ldx, const T* __restrict__ w,
                                                       long long ldw, T* __restrict__ dx, long long lddx,
                                                       float* __restrict__ part, long long rows, int n, int k, int act,
                                                       float slope, int want_w) {
  constexpr int NP = NT * 16, KP = KT * 16, PAD = MatT<T>::PAD, NS = (NP + 31) / 32 * 32;
  typedef T v4 __attribute__((ext_vector_type(4)));
  typedef typename PreT<T>::type preT;
  typedef preT p4 __attribute__((ext_vector_type(4)));
  __shared__ __align__(16) T dz[64 * (NS + PAD)];   // [row][n]
  __shared__ __align__(16) T dzt[NP * (64 + PAD)];  // [n][row]
  __shared__ __align__(16) T xt[KP * (64 + PAD)];   // [k][row]
  __shared__ __align__(16) T wt[KP * (NS + PAD)];   // [k][n]
  __shared__ float red[256 * 4];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, row = lane & 15, g = lane >> 4;
  for (int q = tid; q < KP * NS; q += 256) {
    const int c = q % KP, j = q / KP;
    wt[c * (NS + PAD) + j] = dx && c < k && j < n ? w[(long long)j * ldw + c] : from_f<T>(0.f);
  }
  if constexpr (NS > NP)
    for (int q = tid; q < 64 * (NS - NP); q += 256) dz[q / (NS - NP) * (NS + PAD) + NP + q % (NS - NP)] = from_f<T>(0.f);
  f32x4_m aw[KT] = {};
  f32x4_m sb = {};
  for (long long r0 = blockIdx.x * 64LL; r0 < rows; r0 += gridDim.x * 64LL) {
    constexpr int NC = NP / 4, KC = KP / 4, UN = 64 * NC / 256, UK = 64 * KC / 256;  // chunks of four a row, a thread
    v4 vy[UN], vx[UK];
    p4 vz[UN];
#pragma unroll
    for (int u = 0; u < UN; ++u) {
      const int q = u * 256 + tid, j = q % NC * 4;
      const long long i = r0 + q / NC;
      vy[u] = v4{};
      vz[u] = p4{};
      if (i < rows && j < n) {
        if (j + 4 <= n) {
          vy[u] = load_v<v4>(dy + i * lddy + j);
          if (act != CGAN3D_ACT_NONE) vz[u] = load_v<p4>(pre + i * n + j);
        } else {
#pragma unroll
          for (int r = 0; r < 4; ++r)
            if (j + r < n) {
              vy[u][r] = dy[i * lddy + j + r];
              if (act != CGAN3D_ACT_NONE) vz[u][r] = pre[i * n + j + r];
            }
        }
      }
    }
    if (want_w) {
#pragma unroll
      for (int u = 0; u < UK; ++u) {
        const int q = u * 256 + tid, c = q % KC * 4;
        const long long i = r0 + q / KC;
        vx[u] = v4{};
        if (i < rows && c < k) {
          if (c + 4 <= k) vx[u] = load_v<v4>(x + i * ldx + c);
          else
#pragma unroll
            for (int r = 0; r < 4; ++r)
              if (c + r < k) vx[u][r] = x[i * ldx + c + r];
        }
      }
    }
    __syncthreads();  // the previous tile's fragments are read
#pragma unroll
    for (int u = 0; u < UN; ++u) {
      const int q = u * 256 + tid, j = q % NC * 4, i = q / NC;
      v4 o;
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        float v = to_f(vy[u][r]);
        if (act != CGAN3D_ACT_NONE) v *= mat_act_grad<sizeof(T) == 2>(to_f(vz[u][r]), act, slope);
        sb[r] += v;
        o[r] = from_f<T>(v);
        dzt[(j + r) * (64 + PAD) + i] = o[r];
      }
      *reinterpret_cast<v4*>(&dz[i * (NS + PAD) + j]) = o;
    }
    if (want_w) {
#pragma unroll
      for (int u = 0; u < UK; ++u) {
        const int q = u * 256 + tid, c = q % KC * 4, i = q / KC;
#pragma unroll
        for (int r = 0; r < 4; ++r) xt[(c + r) * (64 + PAD) + i] = vx[u][r];
      }
    }
    __syncthreads();
    if (dx) {  // a wave: 16 rows, every column
      f32x4_m ax[KT] = {};
#pragma unroll
      for (int s = 0; s < NS / 32; ++s)
#pragma unroll
        for (int t = 0; t < KT; ++t)
          ax[t] = mfma_8(&wt[(t * 16 + row) * (NS + PAD) + s * 32 + g * 8], &dz[(wave * 16 + row) * (NS + PAD) + s * 32 + g * 8], ax[t]);
      const long long i = r0 + wave * 16 + row;
      if (i < rows)
#pragma unroll
        for (int t = 0; t < KT; ++t) {
          const int c = t * 16 + g * 4;
          if (c >= k) continue;
          v4 o;
#pragma unroll
          for (int r = 0; r < 4; ++r) o[r] = from_f<T>(ax[t][r]);
          if (c + 4 <= k) store_v(dx + i * lddx + c, o);
          else
#pragma unroll
            for (int r = 0; r < 4; ++r)
              if (c + r < k) dx[i * lddx + c + r] = o[r];
        }
    }
    if (want_w && wave < NT) {  // a wave: 16 rows of dW
#pragma unroll
      for (int s = 0; s < 2; ++s)
#pragma unroll
        for (int t = 0; t < KT; ++t)
          aw[t] = mfma_8(&xt[(t * 16 + row) * (64 + PAD) + s * 32 + g * 8], &dzt[(wave * 16 + row) * (64 + PAD) + s * 32 + g * 8], aw[t]);
    }
  }
  // partial sums: [block][n k + n]
  if (!part) return;
  float* o = part + (long long)blockIdx.x * (n * k + n);
  if (want_w && wave < NT) {
    const int j = wave * 16 + row;
    if (j < n)
#pragma unroll
      for (int t = 0; t < KT; ++t)
#pragma unroll
        for (int r = 0; r < 4; ++r)
          if (t * 16 + g * 4 + r < k) o[j * k + t * 16 + g * 4 + r] = aw[t][r];
  }
  constexpr int NC = NP / 4;
  *reinterpret_cast<f32x4_m*>(red + tid * 4) = sb;
  __syncthreads();
  if (tid < NP && tid < n) {
    float s = 0.f;
    for (int q = tid / 4; q < 256; q += NC) s += red[q * 4 + tid % 4];
    o[n * k + tid] = s;
  }
}

// out[c] = sum of part[b][c] over nb rows of `width`, 16 columns a block, 64 threads on each, added in a fixed order; the
// columns from n k on are db's
template <typename T>
__global__ __launch_bounds__(1024) void rows_join_kernel(const float* __restrict__ part, int nb, int width, int nk,
                                                         T* __restrict__ dw, T* __restrict__ db) {
  __shared__ float red[64][17];
  const int c = threadIdx.x & 15, r = threadIdx.x >> 4, col = blockIdx.x * 16 + c;
  float s = 0.f;
  if (col < width)
#pragma unroll 8
    for (int b = r; b < nb; b += 64) s += part[(long long)b * width + col];
  red[r][c] = s;
  __syncthreads();
  if (r == 0 && col < width) {
    double a = 0.;
    for (int q = 0; q < 64; ++q) a += red[q][c];
    if (col < nk) {
      if (dw) dw[col] = from_f<T>((float)a);
    } else if (db) {
      db[col - nk] = from_f<T>((float)a);
    }
  }
}

bool skinny_takes(const cgan3d_linear_args* a) {
  return a->rows <= kSkinnyRows && (a->dtype == CGAN3D_DT_F32 || a->n <= 32 * cu_count());
}
bool few_channels(long long n, long long k) { return n > 0 && k > 0 && n <= 64 && k <= 64; }
// rows_fwd_kernel against the products' own.  f32 always: 64 rows of 64 -> 64 6.4 / 7.0 us, 16384 7.2 / 7.8, 1048576 148 / 198.
// 16-bit tensors lose with more than two column tiles until there are rows enough, unless the products have to copy
// their operands first: bf16 64 -> 64 512 rows 4.7 / 4.0, 16384 5.0 / 4.3, 131072 15.3 / 12.3, 262144 21.3 / 22.5; 32 -> 64
// 16384 4.9 / 4.3, 65536 6.4 / 7.6; 64 -> 32 4096 3.8 / 4.0; 60 -> 60 4096 5.7 / 6.5.
bool rows_fwd_takes(const cgan3d_linear_args* a) {
  if (!few_channels(a->n, a->k)) return false;
  if (a->dtype == CGAN3D_DT_F32 || a->n <= 32 || !chunked(a->x, a->ldx, a->k) || !chunked(a->w, a->ldw, a->k)) return true;
  return a->rows > (a->k > 48 ? 1 << 17 : 1 << 14);
}
// One pass against dz, two products and their joins.  Always, but for 16-bit tensors of whole chunks with more than two tiles
// each way and an activation, whose few blocks take longer than the products until there are rows enough.  us, 8 / 256
// rows with SiLU: f32 64 -> 64 16.5 / 17.1 and 16.0 / 26.8 (products), 16 -> 64 11.1 / 11.4 and 14.0 / 23.9; bf16 64 -> 64
// 13.5 / 14.3 and 11.9 / 13.6 (512 rows: 14.3 and 15.3), 32 -> 32 9.1 / 9.3 and 12.0 / 13.6, 33 -> 50 12.7 / 14.2 and 15.7 /
// 18.2; without an activation bf16 64 -> 64 11.0 / 11.7 and 11.0 / 12.5.
bool rows_bwd_takes(const cgan3d_linear_args* a) {
  if (!few_channels(a->n, a->k) || a->rows == 0 || !(a->dx || a->dw)) return false;
  const bool quick = a->dtype != CGAN3D_DT_F32 && a->act != CGAN3D_ACT_NONE && a->n > 32 && a->k > 32 && a->n % 8 == 0 &&
                     chunked(a->x, a->ldx, a->k) && chunked(a->w, a->ldw, a->k);
  return !quick || a->rows >= 384;
}
int rows_blocks(const cgan3d_linear_args* a) { return (int)std::min<long long>((a->rows + 63) / 64, kRowsBlocks); }

template <typename T, int NT> void rows_fwd_nt(const MatArgs& p, hipStream_t st) {
  const T* x = static_cast<const T*>(p.a);
  const T* w = static_cast<const T*>(p.b);
  // four waves a block; enough blocks to fill the card, each wave going on from there
  const unsigned blocks = (unsigned)std::min((p.I + 63) / 64, 8LL * cu_count());
  if (p.K <= 32) launch(rows_fwd_kernel<T, NT, 1>, dim3(blocks), dim3(256), 0, st, x, p.lda, w, p.ldb, p.I, (int)p.J, (int)p.K, p.e);
  else launch(rows_fwd_kernel<T, NT, 2>, dim3(blocks), dim3(256), 0, st, x, p.lda, w, p.ldb, p.I, (int)p.J, (int)p.K, p.e);
}
template <typename T> void rows_fwd_run(const MatArgs& p, hipStream_t st) {
  if (p.J <= 16) rows_fwd_nt<T, 1>(p, st);
  else if (p.J <= 32) rows_fwd_nt<T, 2>(p, st);
  else rows_fwd_nt<T, 4>(p, st);
}

template <typename T, int NT, int KT> void rows_bwd_nk(const cgan3d_linear_args* a, float* part, hipStream_t st) {
  typedef typename PreT<T>::type preT;
  launch(rows_bwd_kernel<T, NT, KT>, dim3(rows_blocks(a)), dim3(256), 0, st, static_cast<const T*>(a->dy), (long long)a->lddy,
         static_cast<const preT*>(a->preact), static_cast<const T*>(a->x), (long long)a->ldx, static_cast<const T*>(a->w),
         (long long)a->ldw, static_cast<T*>(a->dx), (long long)a->lddx, part, (long long)a->rows, a->n, a->k, a->act,
         a->slope, a->dw != nullptr ? 1 : 0);
}
template <typename T> void rows_bwd_run(const cgan3d_linear_args* a, void* ws, hipStream_t st) {
  float* part = a->dw || a->dbias ? static_cast<float*>(ws) : nullptr;
  const int nt = a->n <= 16 ? 1 : a->n <= 32 ? 2 : 4, kt = a->k <= 16 ? 1 : a->k <= 32 ? 2 : 4;
#define CG_ROWS(N, K) \
  if (nt == N && kt == K) rows_bwd_nk<T, N, K>(a, part, st);
  CG_ROWS(1, 1) CG_ROWS(1, 2) CG_ROWS(1, 4) CG_ROWS(2, 1) CG_ROWS(2, 2) CG_ROWS(2, 4) CG_ROWS(4, 1) CG_ROWS(4, 2) CG_ROWS(4, 4)
#undef CG_ROWS
  if (part) {
    const int width = a->n * a->k + a->n;
    launch(rows_join_kernel<T>, dim3((width + 15) / 16), dim3(1024), 0, st, (const float*)part, rows_blocks(a), width,
           a->n * a->k, static_cast<T*>(a->dw), static_cast<T*>(a->dbias));
  }
}

// --- dz = dy * act'(z), and its column sums ---
// CT threads of a block along the columns (V values each), the rest along the rows; column sums in 32 bits, of dz
// before its rounding, into part [blockIdx.y][n].  dz goes to rows of ldz values whose padding is zeroed: in the tensors'
// type, or (PL3) split into three planes.  Rounding a 16-bit dz once lets both products read it straight into the
// matrix instructions; a second plane of what is lost would double them (error of a large bf16 step 0.0023, without
// 0.0017).  Bound by memory: 8192 x 8192 bf16 with GELU 90 us, 4.5 TB/s.
template <typename T, bool PL3>
__global__ __launch_bounds__(256) void act_grad_kernel(const T* __restrict__ dy, long long lddy,
                                                       const typename PreT<T>::type* __restrict__ pre, void* __restrict__ dzv,
                                                       int ldz, float* __restrict__ part, long long rows, int n,
                                                       long long chunk, int act, float slope, int ct) {
  constexpr int V = MatT<T>::VEC;
  typedef typename PreT<T>::type preT;
  typedef T vecT __attribute__((ext_vector_type(V)));
  typedef preT vecP __attribute__((ext_vector_type(V)));
  __shared__ float red[256 * V];
  const int c = threadIdx.x % ct, r = threadIdx.x / ct, rt = 256 / ct;
  const int j = (blockIdx.x * ct + c) * V;
  const long long i1 = std::min(rows, ((long long)blockIdx.y + 1) * chunk);
  float s[V] = {};
  if (j < n || (dzv && j < ldz)) {
    for (long long i = (long long)blockIdx.y * chunk + r; i < i1; i += rt) {
      float v[V];
      if (j + V <= n) {
        const vecT y = load_v<vecT>(dy + i * lddy + j);
#pragma unroll
        for (int q = 0; q < V; ++q) v[q] = to_f(y[q]);
        if (act != CGAN3D_ACT_NONE) {
          const vecP z = load_v<vecP>(pre + i * n + j);
#pragma unroll
          for (int q = 0; q < V; ++q) v[q] *= mat_act_grad<sizeof(T) == 2>(to_f(z[q]), act, slope);
        }
      } else {
#pragma unroll
        for (int q = 0; q < V; ++q) {
          v[q] = 0.f;
          if (j + q < n) {
            v[q] = to_f(dy[i * lddy + j + q]);
            if (act != CGAN3D_ACT_NONE) v[q] *= mat_act_grad<sizeof(T) == 2>(to_f(pre[i * n + j + q]), act, slope);
          }
        }
      }
#pragma unroll
      for (int q = 0; q < V; ++q) s[q] += v[q];
      if (!dzv) continue;
      if constexpr (PL3) {
        bf16x4_m h, m, l;
#pragma unroll
        for (int q = 0; q < V; ++q) {
          bf16_t t[3];
          split3(v[q], t);
          h[q] = t[0];
          m[q] = t[1];
          l[q] = t[2];
        }
        bf16_t* d = static_cast<bf16_t*>(dzv) + i * ldz + j;
        *reinterpret_cast<bf16x4_m*>(d) = h;
        *reinterpret_cast<bf16x4_m*>(d + rows * ldz) = m;
        *reinterpret_cast<bf16x4_m*>(d + 2 * rows * ldz) = l;
      } else {
        vecT o;
#pragma unroll
        for (int q = 0; q < V; ++q) o[q] = from_f<T>(v[q]);
        *reinterpret_cast<vecT*>(static_cast<T*>(dzv) + i * ldz + j) = o;
      }
    }
  }
  if (!part) return;
#pragma unroll
  for (int q = 0; q < V; ++q) red[(r * V + q) * ct + c] = s[q];
  __syncthreads();
  for (int u = threadIdx.x; u < ct * V; u += 256) {
    float a = 0.f;
    for (int w = 0; w < rt; ++w) a += red[w * V * ct + u];
    const int col = (blockIdx.x * ct + u % ct) * V + u / ct;
    if (col < n) part[(long long)blockIdx.y * n + col] = a;
  }
}

template <typename T>
__global__ __launch_bounds__(256) void bias_join_kernel(const float* __restrict__ part, int nb, int n, T* __restrict__ db) {
  // 16 columns a block, 16 threads on each, added in a fixed order
  __shared__ double red[16][16];
  const int c = threadIdx.x & 15, r = threadIdx.x >> 4;
  const long long j = long_block() * 16LL + c;
  double s = 0.;
  if (j < n)
    for (int b = r; b < nb; b += 16) s += part[(long long)b * n + j];
  red[r][c] = s;
  __syncthreads();
  if (r == 0 && j < n) {
    for (int q = 1; q < 16; ++q) s += red[q][c];
    db[j] = from_f<T>((float)s);
  }
}

struct ActGrid {
  int ct, bx;
  long long chunk, nb;
};
ActGrid act_grid(const cgan3d_linear_args* a) {
  const int v = a->dtype == CGAN3D_DT_F32 ? 4 : 8;
  ActGrid g;
  const long long width = row_pad(a->n);
  g.ct = 1;
  while (g.ct < 32 && g.ct * v < width) g.ct *= 2;
  g.bx = (int)((width + g.ct * v - 1) / (g.ct * v));
  const long long want = std::max(1LL, 8LL * cu_count() / std::max(1, g.bx));
  g.chunk = std::max((long long)(256 / g.ct), (a->rows + want - 1) / want);
  g.nb = (a->rows + g.chunk - 1) / g.chunk;
  return g;
}

// dz: null where dy itself serves (no activation, rows that the products can read)
template <typename T, bool PL3>
void act_grad_run(const cgan3d_linear_args* a, void* dz, int ldz, float* part, hipStream_t st) {
  const ActGrid g = act_grid(a);
  if (g.nb > 0 && a->n > 0)
    launch(act_grad_kernel<T, PL3>, dim3(g.bx, (unsigned)g.nb), dim3(256), 0, st, static_cast<const T*>(a->dy),
           (long long)a->lddy, static_cast<const typename PreT<T>::type*>(a->preact), dz, ldz, part, (long long)a->rows,
           a->n, g.chunk, a->act, a->slope, g.ct);
  if (a->dbias && a->n > 0)
    launch(bias_join_kernel<T>, long_grid((a->n + 15) / 16, 256), dim3(256), 0, st, (const float*)part, (int)g.nb, a->n,
           static_cast<T*>(a->dbias));
}

struct Bwd {  // the backward pass: dz, and where things lie in its workspace
  bool has_dz, planes3;
  int ldz;
  long long dz, part, mat, total;
  Operand za, zb, x, w;  // dz summed over columns (dx) and over rows (dw)
};
Bwd bwd_layout(const cgan3d_linear_args* a) {
  Bwd w = {};
  const int dt = a->dtype;
  if (rows_bwd_takes(a)) {
    w.total = a->dw || a->dbias ? (long long)rows_blocks(a) * (a->n * a->k + a->n) * 4 : 0;
    return w;
  }
  // dz goes to planes where both products are better off with them: they share the splitting
  w.x = {a->x, a->ldx, a->rows, a->k, true, false};
  w.w = {a->w, a->ldw, a->n, a->k, true, false};
  if (dt == CGAN3D_DT_F32 && a->dx && a->dw && a->rows > 0 && a->n > 0 && a->k > 0) {
    const Operand z = {nullptr, 0, a->rows, a->n, false, true}, zt = {nullptr, 0, a->rows, a->n, true, true};
    w.planes3 = f32_planes(z, w.w, a->rows, a->k, a->n) && f32_planes(zt, w.x, a->n, a->k, a->rows);
  }
  const bool direct = a->act == CGAN3D_ACT_NONE && !w.planes3 && (dt == CGAN3D_DT_F32 || chunked(a->dy, a->lddy, a->n));
  w.has_dz = !direct && (a->dx || a->dw);
  w.ldz = (int)row_pad(a->n);
  long long at = w.has_dz ? up256(a->rows * w.ldz * (w.planes3 ? 6 : dt_bytes(dt))) : 0;
  w.part = at;
  if (a->dbias) at += up256(act_grid(a).nb * a->n * 4);
  w.mat = at;
  const bool pl = w.planes3 || (dt != CGAN3D_DT_F32);
  w.za = {a->dy, a->lddy, a->rows, a->n, false, pl};
  if (w.has_dz) w.za.ld = w.ldz;
  w.zb = w.za;
  w.zb.strided = true;
  const long long m1 = a->dx ? product_bytes(dt, w.za, w.w, a->rows, a->k, a->n) : 0;
  const long long m2 = a->dw ? product_bytes(dt, w.zb, w.x, a->n, a->k, a->rows) : 0;
  w.total = at + std::max(m1, m2);  // the two products run one after the other
  return w;
}

// the forward product's operands, and its workspace
void fwd_operands(const cgan3d_linear_args* a, Operand* x, Operand* w) {
  *x = {a->x, a->ldx, a->rows, a->k, false, false};
  *w = {a->w, a->ldw, a->n, a->k, false, false};
}
long long fwd_bytes(const cgan3d_linear_args* a) {
  if (a->rows <= kGemvRows || skinny_takes(a) || rows_fwd_takes(a)) return 0;
  Operand x, w;
  fwd_operands(a, &x, &w);
  return product_bytes(a->dtype, x, w, a->rows, a->n, a->k);
}

const char* lin_check(const cgan3d_linear_args* a, bool bwd) {
  if (!a) return "null args";
  if (a->dtype < CGAN3D_DT_F32 || a->dtype > CGAN3D_DT_F16) return "unknown dtype";
  if (a->rows < 0 || a->k < 0 || a->n < 0) return "negative size";
  if (a->rows > (1LL << 40) || a->k > 1 << 30 || a->n > 1 << 30) return "size too large";
  const bool fits = bwd ? rows_bwd_takes(a) || ((!a->dx || launchable(a->dtype, a->rows, a->k, a->n)) &&
                                                (!a->dw || launchable(a->dtype, a->n, a->k, a->rows)))
                        : a->rows <= kGemvRows || skinny_takes(a) || rows_fwd_takes(a) ||
                              launchable(a->dtype, a->rows, a->n, a->k);
  if (!fits) return "too many tiles for one launch";
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
  if (at) mat_run<true, true>(p, ws, st);
  else if (bt) mat_run<false, true>(p, ws, st);
  else mat_run<false, false>(p, ws, st);
}

}  // namespace cg

using namespace cg;

extern "C" int64_t cgan3d_linear_fwd_ws_bytes(const cgan3d_linear_args* a) {
  if (const char* e = lin_check(a, false)) {
    set_error("cgan3d_linear_fwd_ws_bytes: %s", e);
    return -1;
  }
  return fwd_bytes(a);
}

extern "C" int cgan3d_linear_fwd(const cgan3d_linear_args* a, void* ws, int64_t ws_bytes, void* stream) try {
  const char* e = lin_check(a, false);
  CG_CHECK_ARG(!e, "cgan3d_linear_fwd: %s", e);
  const long long need = fwd_bytes(a);
  CG_CHECK_ARG(ws_bytes >= need && (need == 0 || (ws && reinterpret_cast<uintptr_t>(ws) % 16 == 0)),
               "cgan3d_linear_fwd: workspace of %lld bytes (16-byte aligned) needed, got %lld", need, (long long)ws_bytes);
  const int b = dt_bytes(a->dtype), pb = pre_bytes(a->dtype);
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
  hipStream_t st = (hipStream_t)stream;
  if (a->rows == 0 || a->n == 0) return CGAN3D_OK;
  if (a->rows <= kGemvRows) {
    if (a->dtype == CGAN3D_DT_F32) gemv_run<float>(p, st);
    else if (a->dtype == CGAN3D_DT_BF16) gemv_run<bf16_t>(p, st);
    else gemv_run<f16_t>(p, st);
  } else if (skinny_takes(a)) {
    if (a->dtype == CGAN3D_DT_F32) skinny_run<float>(p, st);
    else if (a->dtype == CGAN3D_DT_BF16) skinny_run<bf16_t>(p, st);
    else skinny_run<f16_t>(p, st);
  } else if (rows_fwd_takes(a)) {
    if (a->dtype == CGAN3D_DT_F32) rows_fwd_run<float>(p, st);
    else if (a->dtype == CGAN3D_DT_BF16) rows_fwd_run<bf16_t>(p, st);
    else rows_fwd_run<f16_t>(p, st);
  } else {
    Operand x0, w0;
    fwd_operands(a, &x0, &w0);
    product(a->dtype, x0, w0, p, ws, st);
  }
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
                     a->act != CGAN3D_ACT_NONE ? span(a->preact, a->rows, a->n, a->n, pre_bytes(a->dtype)) : Span{0, 0}};
  const Span out[] = {span(a->dx, a->rows, a->k, a->lddx, b), span(a->dw, a->n, a->k, a->k, b),
                      span(a->dbias, 1, a->n, a->n, b)};
  for (int o = 0; o < 3; ++o) {
    for (const Span& s : in) CG_CHECK_ARG(!meet(out[o], s), "cgan3d_linear_bwd: a gradient overlaps an operand");
    for (int q = 0; q < o; ++q) CG_CHECK_ARG(!meet(out[o], out[q]), "cgan3d_linear_bwd: two gradients overlap");
  }
  hipStream_t st = (hipStream_t)stream;
  char* base = static_cast<char*>(ws);
  if (rows_bwd_takes(a)) {
    if (a->dtype == CGAN3D_DT_F32) rows_bwd_run<float>(a, ws, st);
    else if (a->dtype == CGAN3D_DT_BF16) rows_bwd_run<bf16_t>(a, ws, st);
    else rows_bwd_run<f16_t>(a, ws, st);
    CG_LAUNCH_CHECK("cgan3d_linear_bwd");
    return CGAN3D_OK;
  }
  void* dz = l.has_dz ? base + l.dz : nullptr;
  float* part = a->dbias ? reinterpret_cast<float*>(base + l.part) : nullptr;
  if (a->dbias || l.has_dz) {
    if (l.planes3) act_grad_run<float, true>(a, dz, l.ldz, part, st);
    else if (a->dtype == CGAN3D_DT_F32) act_grad_run<float, false>(a, dz, l.ldz, part, st);
    else if (a->dtype == CGAN3D_DT_BF16) act_grad_run<bf16_t, false>(a, dz, l.ldz, part, st);
    else act_grad_run<f16_t, false>(a, dz, l.ldz, part, st);
  }
  MatArgs p = {};
  p.a = l.has_dz ? dz : a->dy;
  p.lda = l.has_dz ? l.ldz : a->lddy;
  p.e.alpha = 1.f;
  if (a->dx) {
    MatArgs q = p;
    Operand z = l.za;
    z.p = p.a;
    q.b = a->w; q.ldb = a->ldw;
    q.I = a->rows; q.J = a->k; q.K = a->n;
    q.e.out = a->dx; q.e.ldo = a->lddx;
    product(a->dtype, z, l.w, q, base + l.mat, st);
  }
  if (a->dw) {
    MatArgs q = p;
    Operand z = l.zb;
    z.p = p.a;
    q.b = a->x; q.ldb = a->ldx;
    q.I = a->n; q.J = a->k; q.K = a->rows;
    q.e.out = a->dw; q.e.ldo = a->k;
    product(a->dtype, z, l.x, q, base + l.mat, st);
  }
  CG_LAUNCH_CHECK("cgan3d_linear_bwd");
  return CGAN3D_OK;
} catch (...) {
  set_error("cgan3d_linear_bwd: out of host memory");
  return CGAN3D_EHIP;
}
