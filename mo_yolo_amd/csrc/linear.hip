// Linear with its epilogue as a trained operator, forward and backward (nn.Linear + activation + residual of the decoder layers' feed-forward
// blocks, nn/modules/transformer.py:515-652, of QIM, MOTR/models/qim.py:73-340, and of the box heads' MLPs, transformer.py:149-161).
//
//   z = x W^T + b    y = act(z) + r          dz = dy act'(z)    dx = dz W    dW = dz^T x    db = sum_rows dz    dr = dy
//
// One matrix-core kernel, C[m, n] = sum_k A[m, k] B[n, k], serves the three products: an operand is either ROW (k contiguous: x, W, dz of dx) or COL (k is
// the row axis in memory: W of dx, dz and x of dW), and COL operands come out of LDS through the transposing read (16-bit) or by single elements (fp32), so
// nothing is transposed in memory.  fp32 products are exact (16x16x4); 16-bit ones run 16x16x32.  Both operands go from memory straight into LDS
// (128 bytes of k to a tile row, XOR-swizzled by way of the lanes' source addresses, what lies outside a matrix arrives as zeros), double-buffered
// with one barrier per tile of k.  Products with too few tiles for the chip are split over k: fp32 partial results, joined in order by a second kernel that
// also runs the epilogue.  Up to 32 rows (a new token of each sequence) take lin_few_kernel, which streams W once through registers.
// dz is its own pass (it feeds two products and the sums of db; in the products' prologues it would be recomputed for every column tile).
// Rows whose length or address is not a whole number of 16-byte steps are copied into padded rows first.
#include "chunk.hpp"

namespace moy {

struct LinParams {
  const void *a, *b;                       // operands: ROW [M or N][K], COL [K][M or N], row strides lda / ldb (elements)
  int64_t lda, ldb;
  int M, N, K;
  const void* bias; int bias_dtype, act;
  const void* r; int64_t ldr;
  void* y; int64_t ldy;
  void* z; int64_t ldz;                    // z as well (NULL: no)
  float* part; int splits, split_tiles;    // split over k: fp32 [splits][M][N], each split_tiles tiles of k
  int tiles_m, tiles_n, vec;               // vec: four neighbouring outputs are one aligned access
};

template <typename T>
struct LFrag {
  u32x4 w;
};
template <>
struct LFrag<float> {
  f32x4 lo, hi;
};
__device__ __forceinline__ f32x4 lin_mma(f32x4 acc, const LFrag<bf16_t>& a, const LFrag<bf16_t>& b) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a.w), __builtin_bit_cast(bf16x8, b.w), acc, 0, 0, 0);
}
__device__ __forceinline__ f32x4 lin_mma(f32x4 acc, const LFrag<f16_t>& a, const LFrag<f16_t>& b) {
  return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a.w), __builtin_bit_cast(f16x8, b.w), acc, 0, 0, 0);
}
__device__ __forceinline__ f32x4 lin_mma(f32x4 acc, const LFrag<float>& a, const LFrag<float>& b) {
#pragma unroll
  for (int e = 0; e < 4; ++e) acc = __builtin_amdgcn_mfma_f32_16x16x4f32(a.lo[e], b.lo[e], acc, 0, 0, 0);
#pragma unroll
  for (int e = 0; e < 4; ++e) acc = __builtin_amdgcn_mfma_f32_16x16x4f32(a.hi[e], b.hi[e], acc, 0, 0, 0);
  return acc;
}

// the activation and its derivative; fp32 by the accurate exponential and quotient, 16-bit types by the fast ones (about 2 ulp of fp32)
template <typename T>
__device__ __forceinline__ float lin_sigmoid(float v) {
  if constexpr (sizeof(T) == 4) return sigmoidf_(v);
  else return fast_sigmoid(v);
}
template <typename T>
__device__ __forceinline__ float lin_act(float v, int act) {
  switch (act) {
    case MOY_ACT_SILU: return v * lin_sigmoid<T>(v);
    case MOY_ACT_RELU: return v < 0.f ? 0.f : v;
    case MOY_ACT_SIGMOID: return lin_sigmoid<T>(v);
    default: return v;
  }
}
template <typename T>
__device__ __forceinline__ float lin_act_grad(float v, int act) {
  const float s = lin_sigmoid<T>(v);
  switch (act) {
    case MOY_ACT_SILU: return s * (1.f + v * (1.f - s));
    case MOY_ACT_RELU: return v > 0.f ? 1.f : v != v ? v : 0.f;
    case MOY_ACT_SIGMOID: return s * (1.f - s);
    default: return 1.f;
  }
}

// four outputs of row m from column n on: bias, z, activation, residual
template <typename T>
__device__ __forceinline__ void lin_finish(const LinParams& p, int m, int n, f32x4 v) {
  if (m >= p.M || n >= p.N) return;
  T* y = static_cast<T*>(p.y) + (int64_t)m * p.ldy + n;
  T* z = p.z ? static_cast<T*>(p.z) + (int64_t)m * p.ldz + n : nullptr;
  const T* r = p.r ? static_cast<const T*>(p.r) + (int64_t)m * p.ldr + n : nullptr;
  if (p.vec) {                             // (N is a multiple of 4 then)
    if (p.bias) v += f32x4{typed_load(p.bias, p.bias_dtype, n), typed_load(p.bias, p.bias_dtype, n + 1), typed_load(p.bias, p.bias_dtype, n + 2),
                           typed_load(p.bias, p.bias_dtype, n + 3)};
    if (z) DT<T>::store4(z, v);
#pragma unroll
    for (int e = 0; e < 4; ++e) v[e] = lin_act<T>(v[e], p.act);
    if (r) v += DT<T>::load4(r);
    DT<T>::store4(y, v);
  } else {
#pragma unroll
    for (int e = 0; e < 4; ++e)
      if (n + e < p.N) {
        float u = v[e] + (p.bias ? typed_load(p.bias, p.bias_dtype, n + e) : 0.f);
        if (z) DT<T>::store1(z + e, u);
        u = lin_act<T>(u, p.act);
        DT<T>::store1(y + e, r ? u + DT<T>::load1(r + e) : u);
      }
  }
}

// 16 bytes for each lane from memory to LDS (wave-uniform LDS base + lane * 16); an offset past the descriptor's range brings zeros.  No register is written; the
// kernel waits on vmcnt itself.
__device__ __forceinline__ void lin_dma16(uint32_t voff, __amdgpu_buffer_rsrc_t rs, uint32_t lds) {
  unsigned keep;
  asm volatile("s_mov_b32 %0, m0\n\ts_mov_b32 m0, %2\n\ts_nop 4\n\tbuffer_load_dwordx4 %1, %3, 0 offen lds\n\ts_mov_b32 m0, %0"
               : "=&s"(keep)
               : "v"(voff), "s"(lds), "s"(rs)
               : "memory");
}

typedef short lin_s16x4 __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) lin_s16x4* lin_lds_s16x4;

// One operand's tile of R rows (of C) by 128 bytes of k (64 elements of 16 bits, 32 of fp32).
//   ROW: LDS [R][8 pieces of 16 bytes], piece c of row r at c ^ ((r >> 1) & 7): a fragment read's 16 rows hit 16 distinct places.
//   COL: LDS [BK][R elements], piece c of k-row r at c ^ (((r & 3) << 1) | (((r >> 3) & 1) << 3)): the transposing read's four rows by two pieces are distinct.
template <typename T, bool COL, int R, int WAVES>
struct LinTile {
  static constexpr int ES = sizeof(T), VEC = 16 / ES, BK = 128 / ES, BYTES = R * 128, N = BYTES / 1024 / WAVES, CPR = R * ES / 16;
  static_assert(N * WAVES * 1024 == BYTES, "whole instructions");
  static __device__ __forceinline__ int swz(int row) {
    if constexpr (COL) return (((row & 3) << 1) | (((row >> 3) & 1) << 3)) & (CPR - 1);
    else return (row >> 1) & 7;
  }
  uint32_t off[N];
  int at[N];                               // ROW: first k element of the lane's piece; COL: its k-row
  __device__ __forceinline__ void init(int64_t ld, int row0, int rows, int wave, int lane) {
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int o = (i * WAVES + wave) * 1024 + lane * 16;
      if constexpr (COL) {
        const int k = o / (R * ES), c = (o % (R * ES)) / 16 ^ swz(k);
        at[i] = k;
        off[i] = row0 + c * VEC < rows ? (uint32_t)((int64_t)k * ld * ES + c * 16) : 0x80000000u;
      } else {
        const int r = o / 128, c = (o % 128) / 16 ^ swz(r);
        at[i] = c * VEC;
        off[i] = row0 + r < rows ? (uint32_t)((int64_t)r * ld * ES + c * 16) : 0x80000000u;
      }
    }
  }
  // base: of the tile's rows at this k; left: elements of k from here on
  __device__ __forceinline__ void issue(const T* base, int left, uint32_t lds, int wave) const {
    const auto rs = __builtin_amdgcn_make_buffer_rsrc(const_cast<T*>(base), 0, 0x7fffffffu, 0x00020000);
#pragma unroll
    for (int i = 0; i < N; ++i) lin_dma16(at[i] < left ? off[i] : 0x80000000u, rs, lds + (i * WAVES + wave) * 1024);
  }
  // the operand of 16 rows from r0 on, k panel kp (32 elements)
  static __device__ __forceinline__ LFrag<T> frag(const unsigned char* lds, int r0, int kp, int lane) {
    const int c = lane & 15, g = lane >> 4;
    if constexpr (!COL) {
      const int r = r0 + c;
      const unsigned char* row = lds + r * 128;
      if constexpr (ES == 2) return LFrag<T>{*reinterpret_cast<const u32x4*>(row + (((kp * 4 + g) ^ swz(r)) << 4))};
      else return LFrag<T>{*reinterpret_cast<const f32x4*>(row + (((2 * g) ^ swz(r)) << 4)), *reinterpret_cast<const f32x4*>(row + (((2 * g + 1) ^ swz(r)) << 4))};
    } else if constexpr (ES == 2) {
      const int k = kp * 32 + g * 8 + (c >> 2), piece = r0 / 8 + ((c & 3) >> 1), half = (c & 1) * 8;
      const unsigned char* p = lds + k * (R * 2) + ((piece ^ swz(k)) << 4) + half;
      const unsigned char* q = lds + (k + 4) * (R * 2) + ((piece ^ swz(k + 4)) << 4) + half;
      const lin_s16x4 x = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lin_lds_s16x4)(const_cast<unsigned char*>(p)));
      const lin_s16x4 y = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lin_lds_s16x4)(const_cast<unsigned char*>(q)));
      const u32x2 u = __builtin_bit_cast(u32x2, x), v = __builtin_bit_cast(u32x2, y);
      return LFrag<T>{u32x4{u.x, u.y, v.x, v.y}};
    } else {
      LFrag<T> f;
      const int piece = (r0 + c) / 4, in = (c & 3) * 4;
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const int k = g * 8 + e;
        const float v = *reinterpret_cast<const float*>(lds + k * (R * 4) + ((piece ^ swz(k)) << 4) + in);
        if (e < 4) f.lo[e] = v;
        else f.hi[e - 4] = v;
      }
      return f;
    }
  }
};

template <typename T, bool ACOL, bool BCOL, int WM, int WN, int MI, int NI>
__global__ __launch_bounds__(WM * WN * 64) void lin_gemm_kernel(const LinParams p) {
  constexpr int WAVES = WM * WN, BM = WM * MI * 16, BN = WN * NI * 16, KP = 4 / (int)sizeof(T);
  using TA = LinTile<T, ACOL, BM, WAVES>;
  using TB = LinTile<T, BCOL, BN, WAVES>;
  constexpr int BK = TA::BK, BUF = TA::BYTES + TB::BYTES;
  extern __shared__ __attribute__((aligned(1024))) unsigned char smem[];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), wm = wave / WN, wn = wave % WN;
  const int c = lane & 15, g = lane >> 4;
  int id = blockIdx.x;
  const int tiles = p.tiles_m * p.tiles_n, split = id / tiles;
  id -= split * tiles;
  {   // the blocks of one XCD take consecutive tiles, and those run down panels of eight column tiles: what they share stays in its L2
    const int qd = tiles >> 3, rm = tiles & 7, x = id & 7;
    id = (x < rm ? x * (qd + 1) : rm * (qd + 1) + (x - rm) * qd) + (id >> 3);
  }
  const int panel = id / (8 * p.tiles_m), in = id - panel * 8 * p.tiles_m, wide = min(8, p.tiles_n - panel * 8);
  const int m0 = in / wide * BM, n0 = (panel * 8 + in % wide) * BN;

  const int nk = (p.K + BK - 1) / BK;
  const int t0 = p.part ? split * p.split_tiles : 0, t1 = p.part ? min(nk, t0 + p.split_tiles) : nk;
  TA ta;
  TB tb;
  ta.init(p.lda, m0, p.M, wave, lane);
  tb.init(p.ldb, n0, p.N, wave, lane);
  const T* ab = static_cast<const T*>(p.a) + (ACOL ? (int64_t)m0 : (int64_t)m0 * p.lda);
  const T* bb = static_cast<const T*>(p.b) + (BCOL ? (int64_t)n0 : (int64_t)n0 * p.ldb);
  const int64_t as = ACOL ? BK * p.lda : BK, bs = BCOL ? BK * p.ldb : BK;
  const uint32_t lds = (uint32_t)reinterpret_cast<uintptr_t>(smem);
  auto issue = [&](int t) {
    const uint32_t to = lds + ((t - t0) & 1) * BUF;
    ta.issue(ab + t * as, p.K - t * BK, to, wave);
    tb.issue(bb + t * bs, p.K - t * BK, to + TA::BYTES, wave);
  };
  f32x4 acc[MI][NI];
#pragma unroll
  for (int i = 0; i < MI; ++i)
#pragma unroll
    for (int j = 0; j < NI; ++j) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};
  if (t0 < t1) issue(t0);
  for (int t = t0; t < t1; ++t) {
    // tile t has landed for every wave, and every wave is done with the buffer that the next one fills
    asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
    __builtin_amdgcn_sched_barrier(0);
    __builtin_amdgcn_s_barrier();
    __builtin_amdgcn_sched_barrier(0);
    if (t + 1 < t1) issue(t + 1);
    const unsigned char* buf = smem + ((t - t0) & 1) * BUF;
#pragma unroll
    for (int kp = 0; kp < KP; ++kp) {
      LFrag<T> fb[NI];
#pragma unroll
      for (int j = 0; j < NI; ++j) fb[j] = TB::frag(buf + TA::BYTES, (wn * NI + j) * 16, kp, lane);
#pragma unroll
      for (int i = 0; i < MI; ++i) {
        const LFrag<T> fa = TA::frag(buf, (wm * MI + i) * 16, kp, lane);
#pragma unroll
        for (int j = 0; j < NI; ++j) acc[i][j] = lin_mma(acc[i][j], fb[j], fa);
      }
    }
    __builtin_amdgcn_sched_barrier(0);
  }
  // Epilogue: 16 rows of the wave at a time by way of its own corner of LDS, so that memory is read and written in whole row pieces
  constexpr int PITCH = NI * 16 + 4, QUADS = NI * 4, ROWS = 64 / QUADS;
  static_assert(WAVES * 16 * PITCH * 4 <= 2 * BUF, "the corners fit the tiles");
  asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");                  // (every wave's reads of the tiles are back)
  __builtin_amdgcn_sched_barrier(0);
  __builtin_amdgcn_s_barrier();
  __builtin_amdgcn_sched_barrier(0);
  float* corner = reinterpret_cast<float*>(smem) + wave * 16 * PITCH;
#pragma unroll
  for (int i = 0; i < MI; ++i) {
#pragma unroll
    for (int j = 0; j < NI; ++j) *reinterpret_cast<f32x4*>(corner + c * PITCH + j * 16 + g * 4) = acc[i][j];
    __builtin_amdgcn_wave_barrier();
#pragma unroll 1
    for (int row = lane / QUADS; row < 16; row += ROWS) {
      const int m = m0 + (wm * MI + i) * 16 + row, n = n0 + wn * NI * 16 + lane % QUADS * 4;
      const f32x4 v = *reinterpret_cast<const f32x4*>(corner + row * PITCH + lane % QUADS * 4);
      if (!p.part) {
        lin_finish<T>(p, m, n, v);
      } else if (m < p.M && n < p.N) {
        float* o = p.part + ((int64_t)split * p.M + m) * p.N + n;
        if (p.N % 4 == 0) {
          *reinterpret_cast<f32x4*>(o) = v;
        } else {
#pragma unroll
          for (int e = 0; e < 4; ++e)
            if (n + e < p.N) o[e] = v[e];
        }
      }
    }
    __builtin_amdgcn_wave_barrier();
  }
}

// the splits of C joined in order, and the epilogue: four outputs to a thread
template <typename T>
__global__ __launch_bounds__(256) void lin_join_kernel(const LinParams p) {
  const int quads = (p.N + 3) / 4;
  const int64_t x = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (x >= (int64_t)p.M * quads) return;
  const int m = (int)(x / quads), n = (int)(x - (int64_t)m * quads) * 4;
  f32x4 v = f32x4{0.f, 0.f, 0.f, 0.f};
  const float* o = p.part + (int64_t)m * p.N + n;
  const int64_t step = (int64_t)p.M * p.N;
  if (p.N % 4 == 0) {
#pragma unroll 4
    for (int s = 0; s < p.splits; ++s) v += *reinterpret_cast<const f32x4*>(o + s * step);
  } else {
    for (int s = 0; s < p.splits; ++s)
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (n + e < p.N) v[e] += o[s * step + e];
  }
  lin_finish<T>(p, m, n, v);
}

// Up to 16 * MI rows: a block takes 16 columns, its eight waves every eighth 128-element piece of k straight from memory in operand order; the waves are
// joined in LDS in wave order.
template <typename T, int MI>
__global__ __launch_bounds__(512) void lin_few_kernel(const LinParams p) {
  constexpr int U = 4;
  __shared__ float sums[8][MI * 16][17];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), c = lane & 15, g = lane >> 4;
  const int n0 = blockIdx.x * 16, n = n0 + c;
  const T* w = static_cast<const T*>(p.b) + (int64_t)n * p.ldb + g * 8;
  const T* x = static_cast<const T*>(p.a) + (int64_t)c * p.lda + g * 8;
  f32x4 acc[MI];
#pragma unroll
  for (int i = 0; i < MI; ++i) acc[i] = f32x4{0.f, 0.f, 0.f, 0.f};
  auto get = [&](const T* q, bool in) {
    LFrag<T> f;
    if constexpr (sizeof(T) == 2) {
      f.w = in ? *reinterpret_cast<const u32x4*>(q) : u32x4{0u, 0u, 0u, 0u};
    } else {                                                                  // (K is a multiple of 4 here, the lane's eight may be half there)
      f.lo = in ? *reinterpret_cast<const f32x4*>(q) : f32x4{0.f, 0.f, 0.f, 0.f};
      f.hi = f32x4{0.f, 0.f, 0.f, 0.f};
    }
    return f;
  };
  for (int k0 = wave * 32 * U; k0 < p.K; k0 += 8 * 32 * U) {
    LFrag<T> fw[U], fx[U][MI];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int k = k0 + u * 32 + g * 8;
      fw[u] = get(w + k0 + u * 32, n < p.N && k < p.K);
      if constexpr (sizeof(T) == 4)
        if (n < p.N && k + 4 < p.K) fw[u].hi = *reinterpret_cast<const f32x4*>(w + k0 + u * 32 + 4);
#pragma unroll
      for (int i = 0; i < MI; ++i) {
        const bool row = i * 16 + c < p.M;
        fx[u][i] = get(x + (int64_t)i * 16 * p.lda + k0 + u * 32, row && k < p.K);
        if constexpr (sizeof(T) == 4)
          if (row && k + 4 < p.K) fx[u][i].hi = *reinterpret_cast<const f32x4*>(x + (int64_t)i * 16 * p.lda + k0 + u * 32 + 4);
      }
    }
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int i = 0; i < MI; ++i) acc[i] = lin_mma(acc[i], fw[u], fx[u][i]);
  }
#pragma unroll
  for (int i = 0; i < MI; ++i)
#pragma unroll
    for (int e = 0; e < 4; ++e) sums[wave][i * 16 + c][g * 4 + e] = acc[i][e];
  __syncthreads();
  for (int t = tid; t < MI * 16 * 4; t += 512) {
    const int m = t >> 2, q = (t & 3) * 4;
    f32x4 v = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int s = 0; s < 8; ++s)
#pragma unroll
      for (int e = 0; e < 4; ++e) v[e] += sums[s][m][q + e];
    lin_finish<T>(p, m, n0 + q, v);
  }
}

// dz = dy act'(z) into rows of `pitch` elements (columns past N: zeros), and the sums of its columns over every gridDim.y-th group of eight rows: a lane
// keeps 16 bytes of columns, the block's eight rows are added in order.  dz NULL: the sums alone; part NULL: dz alone.
template <typename T>
__global__ __launch_bounds__(256) void lin_dz_kernel(const T* __restrict__ dy, int64_t ldd, const T* __restrict__ z, int64_t ldz, int act, int M, int N, T* dz,
                                                     int64_t pitch, float* part) {
  using K = Chunk<T>;
  constexpr int VEC = K::VEC;
  __shared__ float sums[8][32 * VEC + 1];
  const int t = threadIdx.x & 31, rg = threadIdx.x >> 5, n = (blockIdx.x * 32 + t) * VEC;
  float sum[VEC];
#pragma unroll
  for (int e = 0; e < VEC; ++e) sum[e] = 0.f;
  for (int64_t m = (int64_t)blockIdx.y * 8 + rg; m < M; m += (int64_t)gridDim.y * 8) {
    float v[VEC], u[VEC];
    K::load(dy + m * ldd + n, N - n, v);
    if (act != MOY_ACT_NONE) {
      K::load(z + m * ldz + n, N - n, u);
#pragma unroll
      for (int e = 0; e < VEC; ++e) v[e] *= lin_act_grad<T>(u[e], act);        // (past N: 0 times a number)
    }
#pragma unroll
    for (int e = 0; e < VEC; ++e) sum[e] += v[e];
    if (dz && n < pitch) K::store(dz + m * pitch + n, (int)pitch - n, v);
  }
  if (!part) return;
#pragma unroll
  for (int e = 0; e < VEC; ++e) sums[rg][t * VEC + e] = sum[e];
  __syncthreads();
  const int col = threadIdx.x, at = blockIdx.x * 32 * VEC + col;
  if (col < 32 * VEC && at < N) {
    float s = 0.f;
#pragma unroll
    for (int k = 0; k < 8; ++k) s += sums[k][col];
    part[(int64_t)blockIdx.y * N + at] = s;
  }
}

// [rows][n] -> rows of `pitch` elements, zeros behind n
template <typename T>
__global__ __launch_bounds__(256) void lin_pad_kernel(const T* __restrict__ src, int64_t ld, int64_t rows, int n, T* __restrict__ dst, int64_t pitch) {
  using K = Chunk<T>;
  const int64_t chunks = pitch / K::VEC, x = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (x >= rows * chunks) return;
  const int64_t row = x / chunks;
  const int c = (int)(x - row * chunks) * K::VEC;
  float v[K::VEC];
  K::load(src + row * ld + c, n - c, v);
  K::store(dst + row * pitch + c, K::VEC, v);
}

// -------------------------------------------------------------------------------------------------------------------------------- host
struct LinPick {
  int tile;                                // 256, 128 or 64 rows and columns to a block
  int splits, split_tiles;
};

// The largest tile that still gives the chip's 256 compute units a block each, splits of at least four tiles of k counted in (16 at most); 64 otherwise.
static LinPick lin_pick(int M, int N, int K, int es) {
  const int nk = (int)(((int64_t)K * es + 127) / 128);
  for (int tile : {256, 128, 64}) {
    const int64_t tiles = (int64_t)((M + tile - 1) / tile) * ((N + tile - 1) / tile);
    int64_t s = 1;
    if (tiles < 256) {
      s = (512 + tiles - 1) / tiles;
      if (s > nk / 4) s = nk / 4;
      if (s > 16) s = 16;
      if (s < 1) s = 1;
    }
    if (tile == 256 && s > 1) continue;    // (partial results of a split cost more than the larger tile saves)
    if (tiles * s >= 192 || tile == 64) {
      const int per = (int)((nk + s - 1) / s);
      return {tile, (nk + per - 1) / per, per};
    }
  }
  return {64, 1, nk};
}

static int64_t lin_round(int64_t bytes) { return (bytes + 255) / 256 * 256; }
static int lin_es(int dtype) { return dtype == MOY_F32 ? 4 : 2; }
// rows of n elements that the kernels can take as they are
static bool lin_direct(const void* p, int64_t ld, int n, int es) { return aligned16(p) && ld * es % 16 == 0 && (int64_t)n * es % 16 == 0; }
static int64_t lin_pitch(int n, int es) { return ((int64_t)n * es + 15) / 16 * 16 / es; }

static bool lin_few(int M) { return M <= 32; }

template <typename T, bool ACOL, bool BCOL>
static int lin_gemm(LinParams p, float* part, hipStream_t st) {
  const LinPick k = lin_pick(p.M, p.N, p.K, sizeof(T));
  p.tiles_m = (p.M + k.tile - 1) / k.tile;
  p.tiles_n = (p.N + k.tile - 1) / k.tile;
  p.splits = k.splits;
  p.split_tiles = k.split_tiles;
  p.part = k.splits > 1 ? part : nullptr;
  p.vec = p.N % 4 == 0 && p.ldy % 4 == 0 && reinterpret_cast<uintptr_t>(p.y) % (4 * sizeof(T)) == 0 &&
          (!p.z || (p.ldz % 4 == 0 && reinterpret_cast<uintptr_t>(p.z) % (4 * sizeof(T)) == 0)) &&
          (!p.r || (p.ldr % 4 == 0 && reinterpret_cast<uintptr_t>(p.r) % (4 * sizeof(T)) == 0));
  const dim3 grid((unsigned)((int64_t)p.tiles_m * p.tiles_n * k.splits));
#define MOY_LIN(WM, WN, MI, NI)                                                                                                     \
  {                                                                                                                                 \
    auto kern = lin_gemm_kernel<T, ACOL, BCOL, WM, WN, MI, NI>;                                                                     \
    static const bool ready = hipFuncSetAttribute(reinterpret_cast<const void*>(kern), hipFuncAttributeMaxDynamicSharedMemorySize, 160 * 1024) == hipSuccess; \
    if (!ready) return MOY_ELAUNCH;                                                                                                 \
    hipLaunchKernelGGL(kern, grid, dim3(WM * WN * 64), 2 * 128 * (WM * MI * 16 + WN * NI * 16), st, p);                                \
  }
  if (k.tile == 256) MOY_LIN(2, 4, 8, 4)
  else if (k.tile == 128) MOY_LIN(2, 2, 4, 4)
  else MOY_LIN(2, 2, 2, 2)
#undef MOY_LIN
  const int rc = launch_status();
  if (rc != MOY_OK || k.splits == 1) return rc;
  const int64_t quads = (int64_t)p.M * ((p.N + 3) / 4);
  hipLaunchKernelGGL((lin_join_kernel<T>), dim3((unsigned)((quads + 255) / 256)), dim3(256), 0, st, p);
  return launch_status();
}

static int64_t lin_part_bytes(int M, int N, int K, int es) {
  const LinPick k = lin_pick(M, N, K, es);
  return k.splits > 1 ? lin_round((int64_t)k.splits * M * N * 4) : 0;
}

template <typename T>
static int lin_pad(const void* src, int64_t ld, int64_t rows, int n, void* dst, int64_t pitch, hipStream_t st) {
  const int64_t chunks = rows * (pitch / Chunk<T>::VEC);
  hipLaunchKernelGGL((lin_pad_kernel<T>), dim3((unsigned)((chunks + 255) / 256)), dim3(256), 0, st, static_cast<const T*>(src), ld, rows, n, static_cast<T*>(dst), pitch);
  return launch_status();
}

static int lin_check(const moy_linear_args* a, bool bwd) {
  if (!a || a->dtype < MOY_F32 || a->dtype > MOY_F16 || a->M <= 0 || a->N <= 0 || a->K <= 0) return MOY_EINVAL;
  if (a->act < MOY_ACT_NONE || a->act > MOY_ACT_SIGMOID || (a->b_dtype != MOY_F32 && a->b_dtype != a->dtype)) return MOY_EINVAL;
  const int d = a->dtype;
  if (!a->x || !a->w || !aligned_as(a->x, d) || !aligned_as(a->w, d) || (a->M > 1 && a->ldx < 0) || (a->N > 1 && a->ldw < 0)) return MOY_EINVAL;
  if (a->ldx * lin_es(d) > (1 << 22) || a->ldw * lin_es(d) > (1 << 22) || (int64_t)a->K * lin_es(d) > (1 << 22) || (int64_t)a->N * lin_es(d) > (1 << 22)) return MOY_ENOSYS;
  if ((int64_t)((a->M + 63) / 64) * ((a->N + 63) / 64) * 16 > 0x7fffffffLL || (int64_t)((a->M + 63) / 64) * ((a->K + 63) / 64) * 16 > 0x7fffffffLL) return MOY_ENOSYS;
  if ((int64_t)a->M * (a->N > a->K ? a->N : a->K) / 4 / 256 > 0x3fffffffLL) return MOY_ENOSYS;
  if (!bwd) {
    if (!a->y || !aligned_as(a->y, d) || (a->M > 1 && a->ldy < a->N) || !aligned_as(a->b, a->b_dtype)) return MOY_EINVAL;
    if (!aligned_as(a->r, d) || (a->r && a->M > 1 && a->ldr < 0) || !aligned_as(a->z, d)) return MOY_EINVAL;
  } else {
    if (!a->dy || !aligned_as(a->dy, d) || (a->M > 1 && a->ldd < 0) || (!a->dx && !a->dw && !a->db)) return MOY_EINVAL;
    if ((a->act != MOY_ACT_NONE && !a->z) || !aligned_as(a->z, d) || !aligned_as(a->dx, d) || !aligned_as(a->dw, d) || !aligned_as(a->db, a->b_dtype)) return MOY_EINVAL;
    if (a->ldd * lin_es(d) > (1 << 22)) return MOY_ENOSYS;
  }
  return MOY_OK;
}

// What the workspace holds, in this order (bytes, each rounded to 256): padded copies of x and w, dz, the partial results of split products (the largest),
// the partial sums of db.
struct LinPlan {
  bool pad_x, pad_w, make_dz;
  int64_t x, w, dz, part, sums, total;
  int sum_rows;
};
static LinPlan lin_plan(const moy_linear_args* a, bool bwd) {
  const int es = lin_es(a->dtype);
  LinPlan p{};
  p.pad_x = (!bwd || a->dw) && !lin_direct(a->x, a->ldx, a->K, es);
  p.pad_w = (!bwd || a->dx) && !lin_direct(a->w, a->ldw, a->K, es);
  int64_t at = 0;
  p.x = at;
  if (p.pad_x) at += lin_round(a->M * lin_pitch(a->K, es) * es);
  p.w = at;
  if (p.pad_w) at += lin_round(a->N * lin_pitch(a->K, es) * es);
  p.dz = at;
  if (bwd) {
    p.make_dz = (a->dx || a->dw) && (a->act != MOY_ACT_NONE || !lin_direct(a->dy, a->ldd, a->N, es));
    if (p.make_dz) at += lin_round(a->M * lin_pitch(a->N, es) * es);
    p.part = at;
    int64_t most = a->dx ? lin_part_bytes(a->M, a->K, a->N, es) : 0;
    const int64_t other = a->dw ? lin_part_bytes(a->N, a->K, a->M, es) : 0;
    at += most > other ? most : other;
    p.sums = at;
    // about 2048 blocks of the pass over dy, 512 rows of partial sums at most
    const int64_t gx = (a->N + 512 / es - 1) / (512 / es), rows = (a->M + 7) / 8, want = (2048 + gx - 1) / gx;
    p.sum_rows = (int)(rows < want ? rows : want);
    if (p.sum_rows > 512) p.sum_rows = 512;
    if (a->db) at += lin_round((int64_t)p.sum_rows * a->N * 4);
  } else {
    p.part = at;
    if (!lin_few(a->M)) at += lin_part_bytes(a->M, a->N, a->K, es);
  }
  p.total = at;
  return p;
}

template <typename T>
static int lin_fwd(const moy_linear_args* a, const LinPlan& plan, hipStream_t st) {
  char* ws = static_cast<char*>(a->ws);
  const int64_t pitch = lin_pitch(a->K, sizeof(T));
  int rc;
  if (plan.pad_x && (rc = lin_pad<T>(a->x, a->ldx, a->M, a->K, ws + plan.x, pitch, st)) != MOY_OK) return rc;
  if (plan.pad_w && (rc = lin_pad<T>(a->w, a->ldw, a->N, a->K, ws + plan.w, pitch, st)) != MOY_OK) return rc;
  LinParams p{};
  p.a = plan.pad_x ? ws + plan.x : a->x;
  p.lda = plan.pad_x ? pitch : a->ldx;
  p.b = plan.pad_w ? ws + plan.w : a->w;
  p.ldb = plan.pad_w ? pitch : a->ldw;
  p.M = a->M; p.N = a->N;
  p.K = (int)pitch;                        // both rows hold zeros behind K up to a whole 16-byte piece (or K is one already)
  if (!plan.pad_x || !plan.pad_w) p.K = a->K;
  p.bias = a->b; p.bias_dtype = a->b_dtype; p.act = a->act;
  p.r = a->r; p.ldr = a->ldr; p.y = a->y; p.ldy = a->ldy; p.z = a->z; p.ldz = a->N;
  if (lin_few(a->M)) {
    p.vec = p.N % 4 == 0 && p.ldy % 4 == 0 && reinterpret_cast<uintptr_t>(p.y) % (4 * sizeof(T)) == 0 &&
            (!p.z || reinterpret_cast<uintptr_t>(p.z) % (4 * sizeof(T)) == 0) && (!p.r || (p.ldr % 4 == 0 && reinterpret_cast<uintptr_t>(p.r) % (4 * sizeof(T)) == 0));
    const dim3 grid((unsigned)((a->N + 15) / 16));
    if (a->M <= 16) hipLaunchKernelGGL((lin_few_kernel<T, 1>), grid, dim3(512), 0, st, p);
    else hipLaunchKernelGGL((lin_few_kernel<T, 2>), grid, dim3(512), 0, st, p);
    return launch_status();
  }
  return lin_gemm<T, false, false>(p, reinterpret_cast<float*>(ws + plan.part), st);
}

template <typename T>
static int lin_bwd(const moy_linear_args* a, const LinPlan& plan, hipStream_t st) {
  char* ws = static_cast<char*>(a->ws);
  constexpr int ES = sizeof(T);
  const int64_t kp = lin_pitch(a->K, ES), np = lin_pitch(a->N, ES);
  int rc;
  if (plan.pad_x && (rc = lin_pad<T>(a->x, a->ldx, a->M, a->K, ws + plan.x, kp, st)) != MOY_OK) return rc;
  if (plan.pad_w && (rc = lin_pad<T>(a->w, a->ldw, a->N, a->K, ws + plan.w, kp, st)) != MOY_OK) return rc;
  const T* dz = static_cast<const T*>(a->dy);
  int64_t ldz = a->ldd;
  if (plan.make_dz || a->db) {
    T* to = plan.make_dz ? reinterpret_cast<T*>(ws + plan.dz) : nullptr;
    float* sums = a->db ? reinterpret_cast<float*>(ws + plan.sums) : nullptr;
    hipLaunchKernelGGL((lin_dz_kernel<T>), dim3((a->N + 512 / ES - 1) / (512 / ES), plan.sum_rows), dim3(256), 0, st, dz, a->ldd, static_cast<const T*>(a->z),
                       (int64_t)a->N, a->act, a->M, a->N, to, np, sums);
    if ((rc = launch_status()) != MOY_OK) return rc;
    if (sums) {
      hipLaunchKernelGGL(column_sums_kernel, dim3((a->N + 31) / 32), dim3(1024), 0, st, sums, plan.sum_rows, a->N, 0, a->db, static_cast<void*>(nullptr), a->b_dtype);
      if ((rc = launch_status()) != MOY_OK) return rc;
    }
    if (plan.make_dz) {
      dz = to;
      ldz = np;
    }
  }
  float* part = reinterpret_cast<float*>(ws + plan.part);
  if (a->dx) {
    LinParams p{};
    p.a = dz; p.lda = ldz;
    p.b = plan.pad_w ? ws + plan.w : a->w;
    p.ldb = plan.pad_w ? kp : a->ldw;
    p.M = a->M; p.N = a->K; p.K = a->N;
    p.y = a->dx; p.ldy = a->K;
    if ((rc = lin_gemm<T, false, true>(p, part, st)) != MOY_OK) return rc;
  }
  if (a->dw) {
    LinParams p{};
    p.a = dz; p.lda = ldz;
    p.b = plan.pad_x ? ws + plan.x : a->x;
    p.ldb = plan.pad_x ? kp : a->ldx;
    p.M = a->N; p.N = a->K; p.K = a->M;
    p.y = a->dw; p.ldy = a->K;
    if ((rc = lin_gemm<T, true, true>(p, part, st)) != MOY_OK) return rc;
  }
  return MOY_OK;
}

}  // namespace moy

using namespace moy;

extern "C" int64_t moy_linear_ws(const moy_linear_args* a) {
  const int rc = lin_check(a, false);
  return rc != MOY_OK ? rc : lin_plan(a, false).total;
}

extern "C" int moy_linear(const moy_linear_args* a, void* stream) {
  const int64_t need = moy_linear_ws(a);
  if (need < 0) return (int)need;
  if (need > 0 && (!a->ws || !aligned16(a->ws) || a->ws_len < need)) return MOY_EINVAL;
  const LinPlan plan = lin_plan(a, false);
  hipStream_t st = static_cast<hipStream_t>(stream);
  switch (a->dtype) {
    case MOY_F32: return lin_fwd<float>(a, plan, st);
    case MOY_BF16: return lin_fwd<bf16_t>(a, plan, st);
    default: return lin_fwd<f16_t>(a, plan, st);
  }
}

extern "C" int64_t moy_linear_bwd_ws(const moy_linear_args* a) {
  const int rc = lin_check(a, true);
  return rc != MOY_OK ? rc : lin_plan(a, true).total;
}

extern "C" int moy_linear_bwd(const moy_linear_args* a, void* stream) {
  const int64_t need = moy_linear_bwd_ws(a);
  if (need < 0) return (int)need;
  if (need > 0 && (!a->ws || !aligned16(a->ws) || a->ws_len < need)) return MOY_EINVAL;
  const LinPlan plan = lin_plan(a, true);
  hipStream_t st = static_cast<hipStream_t>(stream);
  switch (a->dtype) {
    case MOY_F32: return lin_bwd<float>(a, plan, st);
    case MOY_BF16: return lin_bwd<bf16_t>(a, plan, st);
    default: return lin_bwd<f16_t>(a, plan, st);
  }
}
