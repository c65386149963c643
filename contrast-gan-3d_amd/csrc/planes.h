// Matrix products on 16-bit planes: C[I, J] = sum_t A(i, t) * B(j, t), each operand the sum of P planes.
//
//   P = 1  f16 / bf16 operands as they are
//   P = 2  two f16 planes, hi + lo = 22 bits of a value kept within f16's range by a power of two:
//          hi hi + hi lo + lo hi, three products for f32 accuracy (the Newton-Schulz iteration)
//   P = 3  three bf16 planes, hi + mid + lo = all 24 bits of an f32: the six products of the first two
//          orders (f32 operands of any size; what is left out is below 2^-24 of a product, and of values below 2^-110 what
//          lies under bf16's smallest step, 2^-133)
//
// Bound by the matrix instructions and, there, by the card's power: a Gram product has them busy 68 % of the time at
// 1.63 GHz, a step 42 % at 1.93.  Reached, whole products with their epilogues: P = 1 275 GFLOP (8192 x 8192 -> 2048) in 250
// us, 1100 TFLOP/s; P = 2 the step of two 2048 x 8192 in 381 us, 361 TFLOP/s of f32 accuracy (1082 of 16-bit products);
// P = 3 4096 x 4096 -> 4096 in 677 us with the splitting, 203 TFLOP/s (1218).
// f32 matrix instructions run at 154 TFLOP/s on a large product, 16-bit ones at 1365: a third of that is 455, a
// sixth 227, so f32 accuracy from planes is 3.0 and 1.5 times what the f32 instructions can reach.
//
// A tile's planes go to LDS by DMA (global_load_lds, 16 bytes a lane, one to three stages ahead of the
// products, one barrier a stage).  A t-contiguous operand lies there as rows of BK values and is read by
// ds_read_b128; a t-strided one as BK rows of its own and is read by ds_read_b64_tr_b16, which hands lane i of
// a group of 16 column i of four rows: transposed operands cost no pass over memory.  DMA writes LDS in lane
// order, so bank conflicts are avoided on the global side: each lane fetches the 16-byte chunk whose
// place is its own after an XOR by the row (sw_kc, sw_ks).  Chunks outside the operand come from a zero page.
#pragma once
#include <cmath>

#include "mat.h"

namespace cg {

typedef short s16x4_v __attribute__((ext_vector_type(4)));
typedef short s16x8_v __attribute__((ext_vector_type(8)));

static __device__ __attribute__((aligned(16))) unsigned char g_plane_zero[16];

struct PlaneOp {
  const void* p;    // plane 0
  long long ld;     // elements, a multiple of 8
  long long plane;  // elements between planes
};

// one product; `tiles` x `splits` blocks, split s sums t in [s kchunk, (s + 1) kchunk)
template <class E> struct PlaneJob {
  PlaneOp a, b;
  int I, J, K, tj, tiles, splits, kchunk;
  float* part;  // splits > 1: the tiles' partial sums, [split][tile][BM][BN]
  E e;
};
template <class E, int N> struct PlaneJobs {
  int n;
  int start[N + 1];  // first block of each job
  PlaneJob<E> j[N];
};

// The job of block b: a lane looks at each start, since a trip to the arguments costs about half a microsecond.
template <class E, int N> __device__ __forceinline__ int plane_job(const PlaneJobs<E, N>& jobs, int b) {
  if constexpr (N == 1) return 0;
  const int lane = threadIdx.x & 63;
  return __builtin_amdgcn_readfirstlane(__popcll(__ballot(lane < jobs.n && b >= jobs.start[min(lane, N)])) - 1);
}

// XOR of a chunk's place by its row.  t-contiguous rows of 64 or 128 bytes: 16 lanes read one chunk of 16
// neighbouring rows, which then lie in 16 different 16-byte columns of the 256-byte bank space.  t-strided
// rows: a wave reads 32 bytes of rows 8 g + 4 h + (0..3), g = 0..3: the eight rows of a half wave get eight
// different 32-byte columns (rows of 256 bytes or more; of 128 bytes: four, and the row's own parity).
template <int CH> __device__ __forceinline__ int sw_kc(int r) { return CH == 8 ? (r >> 1) & 7 : -(r >> 2) & 3; }
template <int CH> __device__ __forceinline__ int sw_ks(int k) {
  return CH >= 16 ? 2 * ((k & 3) + 4 * ((k >> 3) & 1)) : 2 * (((k >> 1) & 1) + 2 * ((k >> 3) & 1));
}

// each lane's 16 bytes to lds + 16 * lane; completion is the kernel's own vmcnt wait (the builtin makes
// hipcc count the request on lgkmcnt too, which turns every counted LDS wait into a full one)
__device__ __forceinline__ void plane_dma16(const void* src, unsigned lds) {
  unsigned keep;
  asm volatile("s_mov_b32 %0, m0\n\ts_mov_b32 m0, %2\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, off\n\ts_mov_b32 m0, %0"
               : "=&s"(keep)
               : "v"(src), "s"(lds)
               : "memory");
}

__device__ __forceinline__ f32x4_m plane_mfma(s16x8_v a, s16x8_v b, f32x4_m c, f16_t) {
  return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8_m, a), __builtin_bit_cast(f16x8_m, b), c, 0, 0, 0);
}
__device__ __forceinline__ f32x4_m plane_mfma(s16x8_v a, s16x8_v b, f32x4_m c, bf16_t) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8_m, a), __builtin_bit_cast(bf16x8_m, b), c, 0, 0, 0);
}

// One operand's part of a stage: R rows of the tile (i or j), BK values of t, NW waves.
template <bool KS, int R, int BK, int NW> struct PlaneTile {
  static constexpr int BYTES = R * BK * 2, Q = BYTES / 1024 / NW;  // DMA requests per wave and plane
  static constexpr int CH = KS ? R / 8 : BK / 8;                  // chunks per LDS row
  static_assert(Q >= 1 && BYTES % (1024 * NW) == 0, "whole DMA requests per wave");
  const unsigned short* g[Q];  // this lane's chunk of each request at t = 0
  int kpos[Q];                 // its t within the stage; beyond any K where the chunk is outside the operand

  __device__ __forceinline__ void init(const PlaneOp& o, int n, int r0, int wave, int lane) {
#pragma unroll
    for (int q = 0; q < Q; ++q) {
      const int slot = (q * NW + wave) * 64 + lane, row = slot / CH, pc = slot % CH;
      const unsigned short* p = static_cast<const unsigned short*>(o.p);
      if constexpr (KS) {
        const int col = r0 + (pc ^ sw_ks<CH>(row)) * 8;
        g[q] = p + (long long)row * o.ld + col;
        kpos[q] = col < n ? row : 0x40000000;
      } else {
        const int c = pc ^ sw_kc<CH>(row);
        g[q] = p + (long long)min(r0 + row, n - 1) * o.ld + c * 8;  // rows behind the last: the last one again
        kpos[q] = c * 8;
      }
    }
  }
  // left: t-values from this stage's first to the end
  __device__ __forceinline__ void issue(const PlaneOp& o, long long k, int left, long long plane, unsigned lds, int wave) const {
#pragma unroll
    for (int q = 0; q < Q; ++q) {
      const unsigned short* s = g[q] + (KS ? k * o.ld : k) + plane;
      plane_dma16(kpos[q] < left ? (const void*)s : (const void*)g_plane_zero,
                  __builtin_amdgcn_readfirstlane(lds + (q * NW + wave) * 1024));
    }
  }
};

// Fragment of rows r0 .. + 15 (r0 a multiple of 16), t = 32 s .. + 31 of the stage: lane l gets row l % 16,
// t = (l / 16) * 8 .. + 7.
template <bool KS, int R, int BK>
__device__ __forceinline__ s16x8_v plane_frag(const unsigned char* lds, int r0, int s, int lane) {
  constexpr int CH = KS ? R / 8 : BK / 8;
  if constexpr (KS) {
    const int k = s * 32 + 8 * (lane >> 4) + ((lane & 15) >> 2);
    const int c = (r0 / 8 + ((lane & 3) >> 1)) ^ sw_ks<CH>(k);  // the same for k + 4
    const unsigned char* p = lds + (k * CH + c) * 16 + (lane & 1) * 8;
    typedef __attribute__((address_space(3))) s16x4_v* lp;
    const s16x4_v lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lp)p);
    const s16x4_v hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lp)(p + 4 * CH * 16));
    return __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
  } else {
    const int r = r0 + (lane & 15);
    return *reinterpret_cast<const s16x8_v*>(lds + (r * CH + ((s * 4 + (lane >> 4)) ^ sw_kc<CH>(r))) * 16);
  }
}

// Blocks go to the eight XCDs in turn: give each XCD (its own L2) one run of neighbouring tiles.
__device__ __forceinline__ int xcd_order(int b, int n) {
  const int q = n >> 3, r = n & 7, x = b & 7;
  return x * q + min(x, r) + (b >> 3);
}

template <int BM, bool SYM> __device__ __forceinline__ void plane_tile(int t, int I, int ntj, int& ti, int& tj) {
  if constexpr (SYM) {  // the lower triangle, row after row
    ti = (int)((sqrtf(8.f * t + 1.f) - 1.f) * 0.5f);
    while ((ti + 1) * (ti + 2) / 2 <= t) ++ti;
    while (ti * (ti + 1) / 2 > t) --ti;
    tj = t - ti * (ti + 1) / 2;
  } else {  // columns of eight row tiles: neighbours in time share operand tiles in L2
    constexpr int G = 8;
    const int rows = (I + BM - 1) / BM, g = t / (G * ntj), gr = min(G, rows - g * G), u = t - g * G * ntj;
    ti = g * G + u % gr;
    tj = u / gr;
  }
}

template <int N> __device__ __forceinline__ void wait_vm_only() { asm volatile("s_waitcnt vmcnt(%0)" ::"n"(N) : "memory"); }
template <int N> __device__ __forceinline__ void wait_vm() { asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" ::"n"(N) : "memory"); }

// One BM x BN tile, WI x WJ waves, BK values of t a stage, S stage buffers: S - 1 stages are in flight ahead.
// The barrier that opens a new stage comes before the last row of products of the one before: they cover the
// wait for the other waves and the reads of the next stage's first fragments, each of B's in the registers
// of its predecessor right behind that one's last use.
template <typename T, int P, bool AT, bool BT, int BM, int BN, int BK, int S, int WI, int WJ, bool AHEAD, bool SYM, class E, int N>
__global__ __launch_bounds__(WI * WJ * 64) void plane_kernel(PlaneJobs<E, N> jobs) {
  constexpr int NW = WI * WJ, WM = BM / WI, WN = BN / WJ, FM = WM / 16, FN = WN / 16, H = BK / 32;
  using TA = PlaneTile<AT, BM, BK, NW>;
  using TB = PlaneTile<BT, BN, BK, NW>;
  constexpr int STAGE = P * (TA::BYTES + TB::BYTES), REQ = P * (TA::Q + TB::Q);
  static_assert(S * STAGE <= 160 * 1024 && (S - 1) * REQ < 64, "the stages fit the LDS, their requests the counter");
  static_assert(FM >= 2, "two rows of fragments behind the barrier");
  __shared__ __align__(16) unsigned char lds[S * STAGE];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  int b = xcd_order(blockIdx.x, gridDim.x);
  const int jn = plane_job(jobs, b);
  const PlaneJob<E>& p = jobs.j[jn];
  b -= jobs.start[jn];
  const int split = b / p.tiles, t = b - split * p.tiles;
  int ti, tj;
  plane_tile<BM, SYM>(t, p.I, p.tj, ti, tj);
  const int i0 = ti * BM, j0 = tj * BN;
  const int k0 = split * p.kchunk, k1 = min(p.K, k0 + p.kchunk), steps = (k1 - k0 + BK - 1) / BK;
  const int wi = (wave / WJ) * WM, wj = (wave % WJ) * WN;
  const int own = p.e.begin();  // the epilogue's scalar, on its way under the products

  TA ta;
  TB tb;
  ta.init(p.a, p.I, i0, wave, lane);
  tb.init(p.b, p.J, j0, wave, lane);
  typedef __attribute__((address_space(3))) void* lvp;
  const unsigned base = (unsigned)(uintptr_t)(lvp)lds;
  int slot_in = 0, slot = 0;  // ring positions of the next stage to request and of the one being read
  const auto issue = [&](int s) {
    const int k = k0 + s * BK;
    const unsigned at = base + slot_in * STAGE;
    slot_in = slot_in + 1 == S ? 0 : slot_in + 1;
#pragma unroll
    for (int q = 0; q < P; ++q) {
      ta.issue(p.a, k, k1 - k, q * p.a.plane, at + q * TA::BYTES, wave);
      tb.issue(p.b, k, k1 - k, q * p.b.plane, at + P * TA::BYTES + q * TB::BYTES, wave);
    }
  };
  f32x4_m acc[FM][FN] = {};
  const auto wait_stage = [&](bool all) {  // all but the requests of the S - 2 stages behind
    if (S > 2 && !all) wait_vm<(S - 2) * REQ>();
    else wait_vm<0>();
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
  };
  const auto read_a = [&](s16x8_v(&f)[P], int at, int m, int h) {
    const unsigned char* la = lds + at * STAGE;
#pragma unroll
    for (int q = 0; q < P; ++q) f[q] = plane_frag<AT, BM, BK>(la + q * TA::BYTES, wi + m * 16, h, lane);
  };
  const auto read_b = [&](s16x8_v(&f)[P][FN], int at, int n, int h) {
    const unsigned char* lb = lds + at * STAGE + P * TA::BYTES;
#pragma unroll
    for (int q = 0; q < P; ++q) f[q][n] = plane_frag<BT, BN, BK>(lb + q * TB::BYTES, wj + n * 16, h, lane);
  };
  // small products first; operands swapped, so that a lane ends up with neighbouring columns
  const auto row = [&](int m, const s16x8_v(&a)[P], const s16x8_v(&fb)[P][FN]) {
#pragma unroll
    for (int o = P - 1; o >= 0; --o)
#pragma unroll
      for (int q = 0; q <= o; ++q)
#pragma unroll
        for (int n = 0; n < FN; ++n) acc[m][n] = plane_mfma(fb[o - q][n], a[q], acc[m][n], T());
  };
  if constexpr (AHEAD) {
    // A whole stage of fragments is read a stage ahead: A's each into the registers of the row that has just used
    // them, B's into a second set.  The barrier of stage s finds s + 1 landed and s - 1 read by every wave, and
    // the products behind it need nothing that is not in registers.
    // Stages behind the last are requested and computed too, from the zero page (up to a whole pair): branches
    // would cost more than they save.
    static_assert(H == 1 && S >= 3, "stages: one read late, one being read, one landing");
    s16x8_v fa[FM][P], fb[2][P][FN];
    const auto stage = [&](int s, auto par) {
      constexpr int c = decltype(par)::value;
      wait_vm_only<(S - 3) * REQ>();
      __builtin_amdgcn_s_barrier();
      asm volatile("" ::: "memory");
      issue(s + S - 1);
      slot = slot + 1 == S ? 0 : slot + 1;
#pragma unroll
      for (int m = 0; m < FM; ++m) {
        row(m, fa[m], fb[c]);
        if (m < FN) read_b(fb[c ^ 1], slot, m, 0);
        if (FN > FM && m + FM < FN) read_b(fb[c ^ 1], slot, m + FM, 0);
        read_a(fa[m], slot, m, 0);
      }
    };
#pragma unroll
    for (int s = 0; s < S - 1; ++s) issue(s);
    wait_vm_only<(S - 2) * REQ>();
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
#pragma unroll
    for (int n = 0; n < FN; ++n) read_b(fb[0], 0, n, 0);
#pragma unroll
    for (int m = 0; m < FM; ++m) read_a(fa[m], 0, m, 0);
    int s = 0;
#pragma clang loop unroll(disable)
    do {
      stage(s, std::integral_constant<int, 0>());
      stage(s + 1, std::integral_constant<int, 1>());
      s += 2;
    } while (s < steps);
    wait_vm<0>();  // no request outlives the block
  } else {
    s16x8_v fb[P][FN], fa[2][P];  // B's fragments of the unit, A's first two rows of them
    const auto unit = [&](int s, int h) {
      if (h == 0 && s + S - 1 < steps) issue(s + S - 1);
      s16x8_v fr[FM][P];
#pragma unroll
      for (int m = 0; m < FM - 1; ++m) {
        if (m + 2 < FM) read_a(fr[m + 2], slot, m + 2, h);
        if (m < 2) row(m, fa[m], fb);
        else row(m, fr[m], fb);
      }
      s16x8_v last[P];
#pragma unroll
      for (int q = 0; q < P; ++q) last[q] = FM > 2 ? fr[FM - 1][q] : fa[1][q];
      if (h + 1 == H && s + 1 < steps) {
        wait_stage(s + S - 1 >= steps);
        slot = slot + 1 == S ? 0 : slot + 1;
      }
      // behind the last stage these read that stage again, for nothing: a branch here would cut the row apart
      const int hn = h + 1 < H ? h + 1 : 0;
      read_a(fa[0], slot, 0, hn);
      read_a(fa[1], slot, 1, hn);
#pragma unroll
      for (int n = 0; n < FN; ++n) {  // the last row column by column: its fragment of B is free behind it
#pragma unroll
        for (int o = P - 1; o >= 0; --o)
#pragma unroll
          for (int q = 0; q <= o; ++q) acc[FM - 1][n] = plane_mfma(fb[o - q][n], last[q], acc[FM - 1][n], T());
        read_b(fb, slot, n, hn);
      }
    };
    if (steps > 0) {
#pragma unroll
      for (int s = 0; s < S - 1; ++s)
        if (s < steps) issue(s);
      wait_stage(steps < S - 1);
      read_a(fa[0], 0, 0, 0);
#pragma unroll
      for (int n = 0; n < FN; ++n) read_b(fb, 0, n, 0);
      read_a(fa[1], 0, 1, 0);
      for (int s = 0; s < steps; ++s)
#pragma unroll
        for (int h = 0; h < H; ++h) unit(s, h);
    }
  }
  if (p.part) {
    float* o = p.part + ((long long)split * p.tiles + t) * (BM * BN);
#pragma unroll
    for (int m = 0; m < FM; ++m)
#pragma unroll
      for (int n = 0; n < FN; ++n)
        *reinterpret_cast<f32x4_m*>(o + (wi + m * 16 + (lane & 15)) * BN + wj + n * 16 + (lane >> 4) * 4) = acc[m][n];
    return;
  }
  if constexpr (E::STAGED) {
    // through LDS, a wave's own part of it, so that lanes go along the rows of the output: the epilogue's tensors
    // are read and written in whole lines, and its code is there once per pass and not once per fragment
    constexpr int LD = WN + 4, MB = FM >= 4 && NW * 64 * LD * 4 <= S * STAGE ? 4 : 2, LPR = WN / 4, IT = MB * 16 / (64 / LPR);
    static_assert(NW * MB * 16 * LD * 4 <= S * STAGE && FM % MB == 0 && IT % 4 == 0, "a pass fits the stages' LDS");
    float* my = reinterpret_cast<float*>(lds) + wave * (MB * 16 * LD);
    const int lr = lane / LPR, j = j0 + wj + lane % LPR * 4;
    __syncthreads();  // the last stage's fragments are read
#pragma unroll
    for (int mb = 0; mb < FM; mb += MB) {
#pragma unroll
      for (int m = 0; m < MB; ++m)
#pragma unroll
        for (int n = 0; n < FN; ++n)
          *reinterpret_cast<f32x4_m*>(my + (m * 16 + (lane & 15)) * LD + n * 16 + (lane >> 4) * 4) = acc[mb + m][n];
      asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
      if (j < p.J) {
#pragma clang loop unroll(disable)
        for (int it = 0; it < IT; it += 4) {
          const int r = it * (64 / LPR) + lr;
          f32x4_m v[4];
#pragma unroll
          for (int u = 0; u < 4; ++u) v[u] = *reinterpret_cast<const f32x4_m*>(my + (r + u * (64 / LPR)) * LD + lane % LPR * 4);
          p.e.template put4<64 / LPR>(i0 + wi + mb * 16 + r, j, v, p.I, p.J - j, own);
          if (p.e.turned()) {
#pragma unroll
            for (int u = 0; u < 4; ++u) *reinterpret_cast<f32x4_m*>(my + (r + u * (64 / LPR)) * LD + lane % LPR * 4) = v[u];
          }
        }
      }
      if (p.e.turned()) {  // a transposed output: lanes along its rows, which are the tile's columns
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
        constexpr int LPC = MB * 4;  // lanes per column, four rows each
        const int r = lane % LPC * 4, i = i0 + wi + mb * 16 + r;
        if (i < p.I) {
#pragma clang loop unroll(disable)
          for (int c = lane / LPC; c < WN; c += 64 / LPC) {
            f32x4_m v;
#pragma unroll
            for (int u = 0; u < 4; ++u) v[u] = my[(r + u) * LD + c];
            if (j0 + wj + c < p.J) p.e.put_turned(i, j0 + wj + c, v, p.I - i);
          }
        }
      }
      asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    }
  } else {
#pragma unroll
    for (int m = 0; m < FM; ++m) {
      const int i = i0 + wi + m * 16 + (lane & 15);
      if (i < p.I) {
#pragma unroll
        for (int n = 0; n < FN; ++n) {
          const int j = j0 + wj + n * 16 + (lane >> 4) * 4;
          if (j < p.J) p.e.put(i, j, acc[m][n], p.J - j, SYM && ti != tj, own);
        }
      }
    }
  }
}

// Partial sums added in the order of their splits, then the epilogue: blocks of 16 rows of a tile.
template <int BM, int BN, bool SYM, class E, int N>
__global__ __launch_bounds__(256) void plane_join_kernel(PlaneJobs<E, N> jobs) {
  constexpr int SUB = BM / 16;
  int b = blockIdx.x;
  const int jn = plane_job(jobs, b);
  const PlaneJob<E>& p = jobs.j[jn];
  b -= jobs.start[jn];
  if (!p.part) return;
  const int own = p.e.begin();
  const int t = b / SUB, sub = b - t * SUB;
  int ti, tj;
  plane_tile<BM, SYM>(t, p.I, p.tj, ti, tj);
  bool across = SYM;
  if constexpr (!SYM) across = p.e.turned();
  for (int q = threadIdx.x; q < 16 * BN / 4; q += 256) {
    // lanes along a row; a value that is (also) written to a column: 16 lanes on 16 rows, as the products leave them
    const int li = sub * 16 + (across ? q % 16 : q / (BN / 4)), lj = (across ? q / 16 : q % (BN / 4)) * 4, i = ti * BM + li, j = tj * BN + lj;
    if (i >= p.I || j >= p.J) continue;
    const float* s = p.part + (long long)t * (BM * BN) + li * BN + lj;
    f32x4_m v = *reinterpret_cast<const f32x4_m*>(s);
#pragma unroll 8
    for (int z = 1; z < p.splits; ++z) v += *reinterpret_cast<const f32x4_m*>(s + (long long)z * p.tiles * (BM * BN));
    p.e.put(i, j, v, p.J - j, SYM && ti != tj, own);
  }
}

// --- host side: tiles and splits ---
struct PlaneShape {
  int I, J, K;
};
struct PlanePick {
  int cfg = 0, kchunk = 0;
  long long part_floats = 0;
  double seconds = 0;  // expected
};
// Tile configurations by planes: 0 the largest (8 waves, one block a CU), 1 and 2 smaller ones that give more
// blocks where there are few.  RATE: a CU's share of the largest tile's.  Measured, us, tiles 0 / 1 / 2 without splits and
// what plane_pick took: bf16 8192 x 4096 -> 4096 217 / 310 / 436, took 0; 2048 x 2048 -> 2048 50 / 27 / 36, took 1;
// 512 x 4096 -> 4096 87 / 43 / 34, took 2; f32 the same three 1398 / 1681 / 2465, 154 / 116 / 172 (took 113 with a
// split), 277 / 180 / 162 (140).  Five steps of 4096 x 4096 4412 / 4600 / 6320, took 0 (4305); of 1024 x 4096 1974 / 691 /
// 461, took 406 with splits.
template <int P, bool SYM = false> struct PlaneCfg;
template <> struct PlaneCfg<1, false> {
  static constexpr int BM[3] = {256, 128, 64}, BN[3] = {256, 128, 64}, BK[3] = {32, 32, 64}, WI[3] = {2, 2, 2}, WJ[3] = {4, 2, 2}, S[3] = {5, 5, 4};
  static constexpr bool AHEAD[3] = {true, true, false};
  static constexpr float RATE[3] = {1.f, 0.75f, 0.4f};
};
template <> struct PlaneCfg<2, false> {
  static constexpr int BM[3] = {128, 128, 64}, BN[3] = {256, 128, 64}, BK[3] = {32, 32, 32}, WI[3] = {2, 2, 2}, WJ[3] = {4, 4, 2}, S[3] = {3, 4, 5};
  static constexpr bool AHEAD[3] = {true, true, true};
  static constexpr float RATE[3] = {1.f, 0.8f, 0.5f};
};
template <> struct PlaneCfg<2, true> {
  static constexpr int BM[3] = {256, 128, 64}, BN[3] = {256, 128, 64}, BK[3] = {32, 32, 32}, WI[3] = {2, 2, 2}, WJ[3] = {4, 4, 2}, S[3] = {2, 4, 5};
  static constexpr bool AHEAD[3] = {false, true, true};
  static constexpr float RATE[3] = {1.f, 0.8f, 0.5f};
};
template <> struct PlaneCfg<3, false> {
  static constexpr int BM[3] = {128, 128, 64}, BN[3] = {256, 128, 64}, BK[3] = {32, 32, 32}, WI[3] = {2, 2, 2}, WJ[3] = {4, 4, 2}, S[3] = {2, 3, 4};
  static constexpr bool AHEAD[3] = {false, true, true};
  static constexpr float RATE[3] = {1.f, 0.8f, 0.5f};
};

inline long long plane_tiles(const PlaneShape& s, int bm, int bn, bool sym) {
  const long long ti = ((long long)s.I + bm - 1) / bm, tj = ((long long)s.J + bn - 1) / bn;
  return sym ? ti * (ti + 1) / 2 : ti * tj;
}

// The tile size and the length of a split that the launch of these products is expected to be fastest
// with: the blocks that the fullest CU gets, at the rate a CU reaches with that tile (PlaneCfg::RATE), 64
// t-values' worth of start and end per block, and the joining of partial sums (written and read once, a
// launch of its own).  Measured, us, bf16 128 x 8192 -> 128, tile 2 in 1 / 4 / 16 / 64 splits: 44 / 17 / 12 / 17;
// 128 x 65536 -> 128: 321 / 87 / 30 / 21; 1024 x 16384 -> 1024, tile 1 in 1 / 4 / 16: 140 / 51 / 63, took 53.
template <int P, bool sym> PlanePick plane_pick(const PlaneShape* s, int n) {
  using C = PlaneCfg<P, sym>;
  const double cus = cu_count(), rate = 1.1e15 / (P * (P + 1) / 2) / 2 / cus;  // products of a CU per second
  PlanePick best;
  double tb = 1e30;
  int kmax = 1;
  for (int i = 0; i < n; ++i) kmax = std::max(kmax, s[i].K);
  for (int c = 0; c < 3; ++c) {
    int last = 0;
    for (int sp = 1; sp <= 64; ++sp) {
      const int kc = ((kmax + sp - 1) / sp + 63) / 64 * 64;
      if (kc == last) continue;
      last = kc;
      double blocks = 0;
      long long part = 0;
      for (int i = 0; i < n; ++i) {
        const long long t = plane_tiles(s[i], C::BM[c], C::BN[c], sym), z = std::max(1, (s[i].K + kc - 1) / kc);
        blocks += (double)t * z;
        if (z > 1) part += t * z * C::BM[c] * C::BN[c];
      }
      const double rounds = blocks <= cus ? 1. : std::max(std::ceil(blocks / cus), 1.);
      double t = rounds * C::BM[c] * C::BN[c] * (double)(kc + 64) / (rate * C::RATE[c]);
      if (part) t += part * 8. / 3.5e12 + 4e-6 + sp * 5e-8;
      if (t < tb) {
        tb = t;
        best.cfg = c;
        best.kchunk = kc;
        best.part_floats = part;
        best.seconds = t;
      }
      if (kc <= 128 || blocks >= 2 * cus) break;
    }
  }
  return best;
}

// Fills in tiles, splits, partial sums and block numbers (a, b, I, J, K and e are the caller's), and launches.
template <typename T, int P, bool AT, bool BT, bool SYM, class E, int N>
void plane_run(PlaneJobs<E, N>& jobs, const PlanePick& pick, float* part, hipStream_t st) {
  using C = PlaneCfg<P, SYM>;
  const auto go = [&](auto cfg) {
    constexpr int c = decltype(cfg)::value, BM = C::BM[c], BN = C::BN[c];
    int at = 0, jat = 0;
    bool join = false;
    PlaneJobs<E, N> js = jobs;
    for (int i = 0; i < jobs.n; ++i) {
      PlaneJob<E>& j = jobs.j[i];
      j.tj = (j.J + BN - 1) / BN;
      j.tiles = (int)plane_tiles({j.I, j.J, j.K}, BM, BN, SYM);
      j.kchunk = pick.kchunk;
      j.splits = std::max(1, (j.K + pick.kchunk - 1) / pick.kchunk);
      j.part = j.splits > 1 ? part : nullptr;
      if (j.part) part += (long long)j.tiles * j.splits * BM * BN, join = true;
      js.j[i] = j;
      jobs.start[i] = at;
      js.start[i] = jat;
      at += j.tiles * j.splits;
      jat += j.tiles * (BM / 16);
    }
    if (at == 0) return;
    launch(plane_kernel<T, P, AT, BT, BM, BN, C::BK[c], C::S[c], C::WI[c], C::WJ[c], C::AHEAD[c], SYM, E, N>, dim3(at),
           dim3(C::WI[c] * C::WJ[c] * 64), 0, st, jobs);
    if (join) launch(plane_join_kernel<BM, BN, SYM, E, N>, dim3(jat), dim3(256), 0, st, js);
  };
  if (pick.cfg == 0) go(std::integral_constant<int, 0>());
  else if (pick.cfg == 1) go(std::integral_constant<int, 1>());
  else go(std::integral_constant<int, 2>());
}

// f32 accuracy in planes.  Three bf16: what rounding to nearest leaves is exact, and a value too large to
// round up to a finite bf16 is cut instead.  A value that is not finite goes into the first plane alone.
__device__ __forceinline__ void split3(float x, bf16_t* o) {
  bf16_t h = (bf16_t)x;
  const float inf = __builtin_inff();
  if (fabsf(x) < inf && fabsf((float)h) == inf)
    h = __builtin_bit_cast(bf16_t, (unsigned short)(__float_as_uint(x) >> 16));
  const float r = fabsf(x) < inf ? x - (float)h : 0.f;
  const bf16_t m = (bf16_t)r;
  o[0] = h;
  o[1] = m;
  o[2] = (bf16_t)(r - (float)m);
}
// Two f16.  x is one value from here on: where it is a product or a sum, the compiler else rounds it to f16 once straight
// from its operands (v_fma_mix) and once by way of f32, and the two planes belong to unlike first planes wherever
// the roundings differ (one in 2^13, by 2^-11: ten times the error of a whole iteration).
__device__ __forceinline__ void split2(float x, f16_t* o) {
  asm("" : "+v"(x));
  o[0] = (f16_t)x;
  o[1] = (f16_t)(x - (float)o[0]);
}

}  // namespace cg
