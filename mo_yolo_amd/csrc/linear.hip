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
// also runs the epilogue.  Few rows (a new token of each sequence) take lin_few_kernel, which streams W once through registers.
// Measured (a trace's best and median): 8192 x 4096 -> 4096 bf16 forward with z and a residual 252 to 279 us, dx 231 to 258, dW 224 to 249 (1.09, 1.19 and 1.23 PFLOP/s at best, a
// large library product 1.22); 4800 x 256 -> 1024 14.6, 12, 10 + 4; 1803 x 514 -> 770 fp32 35, 32 + 9, 28 + 5; 4096 x 2048 -> 2048 fp32 320, 334, 356 (0.11 PFLOP/s, the library 0.14);
// one row of 1024 -> 4096 4.7, fp32 6.7: bound by the matrix cores' feeding, launches, the fp32 matrix rate, the trip to memory.
// dz is its own pass (it feeds two products and the sums of db; in the products' prologues it would be recomputed for every column tile).
// In 16-bit types z is kept, and dz enters its products, rounded to T once, which the matrix cores ask of an operand: gradients of SiLU at the large size are 2.4e-3 off in norm, where
// the rounding of an exact result alone makes 1.7e-3; a second operand with what the rounding leaves out would make it that, for twice the matrix work of dx and dW (some 480 us of 721).
// Without an activation, and for ReLU, nothing is rounded but the results.  A z off by half a step moves a derivative by up to that step's size relative to itself (SiLU and sigmoid at
// 10 in bf16: 4 %, of a derivative of 5e-4 and less).  db is summed before dz is rounded.  Who wants neither rounding computes in fp32.
// Loads are 16 bytes from any dword on; where a row ends inside one, the tail is cleared in LDS.  16-bit rows of odd length or at odd elements are
// copied into padded rows first.
#include <type_traits>

#include "chunk.hpp"

namespace moy {

struct LinParams {
  const void *a, *b;                       // operands: ROW [M or N][K], COL [K][M or N], row strides lda / ldb (elements)
  int64_t lda, ldb;
  int64_t a_bytes, b_bytes;                // from the first element to the last one's end
  int M, N, K;
  const void* bias; int bias_dtype, act;
  const void* r; int64_t ldr;
  void* y; int64_t ldy;
  void* z; int64_t ldz;                    // z as well (NULL: no)
  float* part; int splits, split_tiles;    // split over k: fp32 [splits][M][N], each split_tiles tiles of k
  int tiles_m, tiles_n, vec;               // vec: four neighbouring outputs are one aligned access
  int clamp;                               // a row of an operand is no whole number of 16-byte pieces
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

// An argument of the activation as it is kept for the backward: what is finite stays finite and what is not 0 stays on its side of 0 when it is rounded to T.  (fp16
// would hold 7e4 as infinity, where the derivative of SiLU is 0 * infinity, and 2^-26 as 0, where ReLU's gate is shut.)
template <typename T>
__device__ __forceinline__ float lin_kept(float v) {
  if constexpr (sizeof(T) == 4) return v;
  constexpr bool HALF = DT<T>::code == MOY_F16;
  constexpr float MOST = HALF ? 65504.f : 0x1.fep127f;
  if constexpr (HALF) v = fabsf(v) <= 0x1p-25f && v != 0.f ? copysignf(0x1p-24f, v) : v;   // half of the smallest number would still round to 0
  return fabsf(v) < INFINITY ? __builtin_amdgcn_fmed3f(v, -MOST, MOST) : v;
}
template <typename T>
__device__ __forceinline__ f32x4 lin_kept4(f32x4 v) {
#pragma unroll
  for (int e = 0; e < 4; ++e) v[e] = lin_kept<T>(v[e]);
  return v;
}

// the bias of columns n .. n + 3 (zeros without one)
__device__ __forceinline__ f32x4 lin_bias(const LinParams& p, int n) {
  f32x4 b = f32x4{0.f, 0.f, 0.f, 0.f};
  if (p.bias) {
#pragma unroll
    for (int e = 0; e < 4; ++e)
      if (n + e < p.N) b[e] = typed_load(p.bias, p.bias_dtype, n + e);
  }
  return b;
}

// four outputs of row m from column n on, their bias added: z, activation, residual (r: loaded ahead where outputs are whole vectors)
template <typename T>
__device__ __forceinline__ void lin_finish_vec(const LinParams& p, int m, int n, f32x4 v, f32x4 r) {
  if (p.z) DT<T>::store4(static_cast<T*>(p.z) + (int64_t)m * p.ldz + n, lin_kept4<T>(v));
  if (p.act != MOY_ACT_NONE) {
#pragma unroll
    for (int e = 0; e < 4; ++e) v[e] = lin_act<T>(v[e], p.act);
  }
  DT<T>::store4(static_cast<T*>(p.y) + (int64_t)m * p.ldy + n, p.r ? v + r : v);
}
template <typename T>
__device__ __forceinline__ void lin_finish_each(const LinParams& p, int m, int n, f32x4 v) {
#pragma unroll 1
  for (int e = 0; e < 4; ++e) {
    if (n + e >= p.N) break;
    float u = e == 0 ? v.x : e == 1 ? v.y : e == 2 ? v.z : v.w;
    const int64_t at = (int64_t)m * p.ldy + n + e;
    if (p.z) DT<T>::store1(static_cast<T*>(p.z) + (int64_t)m * p.ldz + n + e, lin_kept<T>(u));
    u = lin_act<T>(u, p.act);
    if (p.r) u += DT<T>::load1(static_cast<const T*>(p.r) + (int64_t)m * p.ldr + n + e);
    DT<T>::store1(static_cast<T*>(p.y) + at, u);
  }
}
template <typename T>
__device__ __forceinline__ f32x4 lin_residual(const LinParams& p, int m, int n) {
  return p.r ? DT<T>::load4(static_cast<const T*>(p.r) + (int64_t)m * p.ldr + n) : f32x4{0.f, 0.f, 0.f, 0.f};
}
template <typename T>
__device__ __forceinline__ void lin_finish(const LinParams& p, int m, int n, f32x4 v) {
  if (m >= p.M || n >= p.N) return;
  v += lin_bias(p, n);
  if (p.vec) lin_finish_vec<T>(p, m, n, v, lin_residual<T>(p, m, n));
  else lin_finish_each<T>(p, m, n, v);
}

// the activation on four values, its choice taken once
template <typename T>
__device__ __forceinline__ f32x4 lin_act4(f32x4 v, int act) {
  if (act == MOY_ACT_RELU) {
#pragma unroll
    for (int e = 0; e < 4; ++e) v[e] = v[e] < 0.f ? 0.f : v[e];
  } else if (act != MOY_ACT_NONE) {
    const f32x4 u = v;
#pragma unroll
    for (int e = 0; e < 4; ++e) v[e] = lin_sigmoid<T>(v[e]);
    if (act == MOY_ACT_SILU) v = u * v;
  }
  return v;
}

// Quads of a matrix from row m0, column n0 on; a lane that is not `in` reads zeros and writes nothing.
template <typename T>
struct Out {
  __amdgpu_buffer_rsrc_t rs;
  int64_t pitch;
  __device__ __forceinline__ Out(const void* p, int64_t ld, int m0, int n0) : pitch(ld * (int)sizeof(T)) {
    rs = __builtin_amdgcn_make_buffer_rsrc(const_cast<T*>(static_cast<const T*>(p) + m0 * ld + n0), 0, 0x7fffffffu, 0x00020000);
  }
  __device__ __forceinline__ uint32_t at(int row, int quad, bool in) const { return in ? (uint32_t)(row * (int)pitch + quad * 4 * (int)sizeof(T)) : 0x80000000u; }
  __device__ __forceinline__ void store4(int row, int quad, bool in, f32x4 v) const {
    if constexpr (sizeof(T) == 4) __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(u32x4, v), rs, at(row, quad, in), 0, 0);
    else __builtin_amdgcn_raw_buffer_store_b64(u32x2{DT<T>::pack2(v.x, v.y), DT<T>::pack2(v.z, v.w)}, rs, at(row, quad, in), 0, 0);
  }
  __device__ __forceinline__ f32x4 load4(int row, int quad, bool in) const {
    if constexpr (sizeof(T) == 4) {
      return __builtin_bit_cast(f32x4, __builtin_amdgcn_raw_buffer_load_b128(rs, at(row, quad, in), 0, 0));
    } else {
      const u32x2 w = __builtin_bit_cast(u32x2, __builtin_amdgcn_raw_buffer_load_b64(rs, at(row, quad, in), 0, 0));
      const uint32_t a = w.x, b = w.y;
      return f32x4{DT<T>::lo(a), DT<T>::hi(a), DT<T>::lo(b), DT<T>::hi(b)};
    }
  }
};

// 16 bytes for each lane from memory to LDS (wave-uniform LDS base + lane * 16); an offset past the descriptor's range brings zeros.  No register is written; the
// kernel waits on vmcnt itself.
// The first one waits out a descriptor that vector code may have written (the compiler does not see into the block).
template <bool FIRST>
__device__ __forceinline__ void lin_dma16(uint32_t voff, __amdgpu_buffer_rsrc_t rs, uint32_t lds) {
  if constexpr (FIRST) asm volatile("s_mov_b32 m0, %1\n\ts_nop 4\n\tbuffer_load_dwordx4 %0, %2, 0 offen lds" ::"v"(voff), "s"(lds), "s"(rs) : "memory", "m0");
  else asm volatile("s_mov_b32 m0, %1\n\ts_nop 0\n\tbuffer_load_dwordx4 %0, %2, 0 offen lds" ::"v"(voff), "s"(lds), "s"(rs) : "memory", "m0");
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
  // base: of the tile's rows at this k; range: bytes from there to the operand's end (the hardware clamps by dwords); left: elements of k from here on (0: a
  // tile of zeros, which keeps the count of loads in flight)
  __device__ __forceinline__ void issue(const T* base, uint32_t range, int left, uint32_t lds, int wave) const {
    const auto rs = __builtin_amdgcn_make_buffer_rsrc(const_cast<T*>(base), 0, range, 0x00020000);
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const uint32_t o = at[i] < left ? off[i] : 0x80000000u, to = lds + (i * WAVES + wave) * 1024;
      if (i == 0) lin_dma16<true>(o, rs, to);
      else lin_dma16<false>(o, rs, to);
    }
  }
  // a landed ROW tile whose rows end inside a 16-byte piece: what stands behind the row's `left` elements is cleared
  static __device__ __forceinline__ void clear_tail(unsigned char* lds, int left, int tid, int threads) {
    if constexpr (!COL) {
      const int c = left / VEC, e0 = left % VEC;
      for (int r = tid; r < R; r += threads) {
        T* p = reinterpret_cast<T*>(lds + r * 128 + ((c ^ swz(r)) << 4));
        for (int e = e0; e < VEC; ++e) DT<T>::store1(p + e, 0.f);
      }
    }
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

template <int N>
__device__ __forceinline__ void lin_landed() {
  asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" ::"n"(N) : "memory");
  __builtin_amdgcn_sched_barrier(0);
  __builtin_amdgcn_s_barrier();
  __builtin_amdgcn_sched_barrier(0);
}

template <typename T, bool ACOL, bool BCOL, int WM, int WN, int MI, int NI, int STAGES>
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
  // A 16-byte piece reaches past the operand's end only where a row is no whole number of pieces: elsewhere the range is left wide (p.clamp)
  int64_t a_left = p.a_bytes - (reinterpret_cast<const char*>(ab) - static_cast<const char*>(p.a)) - t0 * as * (int64_t)sizeof(T);
  int64_t b_left = p.b_bytes - (reinterpret_cast<const char*>(bb) - static_cast<const char*>(p.b)) - t0 * bs * (int64_t)sizeof(T);
  ab += t0 * as;
  bb += t0 * bs;
  int left = p.K - t0 * BK;
  if (t0 >= t1) left = 0;
  int more = t1 - t0;                                                          // tiles that are still to be fetched
  const uint32_t lds = (uint32_t)reinterpret_cast<uintptr_t>(smem);
  auto issue = [&](int slot) {
    const uint32_t to = lds + slot * BUF;
    uint32_t ra = 0x7fffffffu, rb = 0x7fffffffu;
    if (p.clamp) {
      ra = a_left < 0 ? 0u : a_left < 0x7fffffff ? (uint32_t)a_left : 0x7fffffffu;
      rb = b_left < 0 ? 0u : b_left < 0x7fffffff ? (uint32_t)b_left : 0x7fffffffu;
      a_left -= as * (int64_t)sizeof(T);
      b_left -= bs * (int64_t)sizeof(T);
    }
    const int have = more > 0 ? left : 0;
    ta.issue(ab, ra, have, to, wave);
    tb.issue(bb, rb, have, to + TA::BYTES, wave);
    ab += as;
    bb += bs;
    left -= BK;
    --more;
  };
  f32x4 acc[MI][NI];
#pragma unroll
  for (int i = 0; i < MI; ++i)
#pragma unroll
    for (int j = 0; j < NI; ++j) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};
  // STAGES buffers: STAGES - 1 tiles are on their way ahead of the one in the matrix cores
#pragma unroll
  for (int x = 0; x < STAGES - 1; ++x) issue(x);
  int slot = 0;
  for (int t = t0; t < t1; ++t) {
    // tile t has landed for every wave, and every wave is done with the buffer that is filled next
    lin_landed<(STAGES - 2) * (TA::N + TB::N)>();
    unsigned char* buf = smem + slot * BUF;
    const int next = slot == 0 ? STAGES - 1 : slot - 1;
    slot = slot == STAGES - 1 ? 0 : slot + 1;
    if (t == nk - 1 && p.K % TA::VEC) {
      TA::clear_tail(buf, p.K - t * BK, tid, WAVES * 64);
      TB::clear_tail(buf + TA::BYTES, p.K - t * BK, tid, WAVES * 64);
      lin_landed<63>();                                                        // (the loads in flight stay in flight)
    }
    // the first panel's operands are on their way out of LDS while the next tile's loads are issued, each further panel's while the one before is multiplied
    LFrag<T> fa[KP][MI], fb[KP][NI];
    auto read = [&](int kp) {
#pragma unroll
      for (int j = 0; j < NI; ++j) fb[kp][j] = TB::frag(buf + TA::BYTES, (wn * NI + j) * 16, kp, lane);
#pragma unroll
      for (int i = 0; i < MI; ++i) fa[kp][i] = TA::frag(buf, (wm * MI + i) * 16, kp, lane);
    };
    read(0);
    issue(next);
#pragma unroll
    for (int kp = 0; kp < KP; ++kp) {
      if (kp + 1 < KP) read(kp + 1);
#pragma unroll
      for (int i = 0; i < MI; ++i)
#pragma unroll
        for (int j = 0; j < NI; ++j) acc[i][j] = lin_mma(acc[i][j], fb[kp][j], fa[kp][i]);
    }
    __builtin_amdgcn_sched_barrier(0);
  }
  // Epilogue: H * 16 rows of the wave at a time by way of its own corner of LDS (quads at quad ^ row: no conflicts either way), so that memory is read and
  // written in whole row pieces, and by a loop whose code is small: every block meets it once, cold.
  constexpr int QUADS = NI * 4, ROWS = 64 / QUADS, H = MI < 4 ? MI : 4;
  static_assert(WAVES * H * 16 * NI * 16 * 4 <= STAGES * BUF, "the corners fit the tiles");
  lin_landed<0>();                                                             // every wave's reads of the tiles are back, no load is on its way
  float* corner = reinterpret_cast<float*>(smem) + wave * H * 16 * NI * 16;
  const int row0 = lane / QUADS, quad = lane % QUADS, n = n0 + wn * NI * 16 + quad * 4;
  const bool inside = n < p.N;
  const f32x4 bias = p.part ? f32x4{0.f, 0.f, 0.f, 0.f} : lin_bias(p, n);
  const bool whole = p.part ? p.N % 4 == 0 : p.vec;                            // four neighbours are one access
  // Whole quads go by descriptors whose range drops what lies outside C: no branch, so that a wait for a residual never waits for the stores behind it.
  // A residual is fetched four row pieces ahead.
  const int mw = m0 + wm * MI * 16, nw = n0 + wn * NI * 16;                    // the wave's corner of C
  Out<T> oy(p.y, p.ldy, mw, nw), oz(p.z, p.ldz, mw, nw), orr(p.r, p.ldr, mw, nw);
  Out<float> op(p.part ? p.part + (int64_t)split * p.M * p.N : nullptr, p.N, mw, nw);
#pragma unroll
  for (int half = 0; half < MI / H; ++half) {
#pragma unroll
    for (int i = 0; i < H; ++i)
#pragma unroll
      for (int j = 0; j < NI; ++j)
        *reinterpret_cast<f32x4*>(corner + (i * 16 + c) * (NI * 16) + (((j * 4 + g) ^ (c & (QUADS - 1))) << 2)) = acc[half * H + i][j];
    __builtin_amdgcn_wave_barrier();
    const int down = half * H * 16 + row0;                                     // the lane's first row below the wave's corner
    auto value = [&](int x) {                                                  // x rows further down
      const int row = row0 + x;
      return *reinterpret_cast<const f32x4*>(corner + row * (NI * 16) + ((quad ^ (row & (QUADS - 1))) << 2)) + bias;
    };
    auto there = [&](int x) { return inside && mw + down + x < p.M; };
    auto rows = [&](auto res) {
      constexpr bool RES = decltype(res)::value;
      f32x4 r[4];
      if constexpr (RES) {
#pragma unroll
        for (int k = 0; k < 4; ++k) r[k] = orr.load4(down + k * ROWS, quad, there(k * ROWS));
      }
#pragma unroll 1
      for (int x = 0; x < H * 16; x += 4 * ROWS) {
        f32x4 now[4];
        if constexpr (RES) {
#pragma unroll
          for (int k = 0; k < 4; ++k) now[k] = r[k];
#pragma unroll
          for (int k = 0; k < 4; ++k) r[k] = orr.load4(down + x + (4 + k) * ROWS, quad, x + (4 + k) * ROWS < H * 16 && there(x + (4 + k) * ROWS));
        }
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          f32x4 v = value(x + k * ROWS);
          const bool in = there(x + k * ROWS);
          if (p.z) oz.store4(down + x + k * ROWS, quad, in, lin_kept4<T>(v));
          v = lin_act4<T>(v, p.act);
          if constexpr (RES) v += now[k];
          oy.store4(down + x + k * ROWS, quad, in, v);
        }
      }
    };
    static_assert(H * 16 % (4 * ROWS) == 0, "whole steps");
    if (p.part && whole) {
#pragma unroll 2
      for (int x = 0; x < H * 16; x += ROWS) op.store4(down + x, quad, there(x), value(x));
    } else if (whole && p.r) {
      rows(std::true_type{});
    } else if (whole) {
      rows(std::false_type{});
    } else if (inside) {
#pragma unroll 1
      for (int x = 0; x < H * 16 && there(x); x += ROWS) {
        const f32x4 v = value(x);
        if (p.part) {
          float* o = p.part + ((int64_t)split * p.M + mw + down + x) * p.N + n;
#pragma unroll
          for (int e = 0; e < 4; ++e)
            if (n + e < p.N) o[e] = v[e];
        } else {
          lin_finish_each<T>(p, mw + down + x, n, v);
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
  // eight elements at any alignment, `left` of them there
  auto get = [&](const T* q, int left) {
    LFrag<T> f;
    if (left >= 8) {
      __builtin_memcpy(&f, __builtin_assume_aligned(q, sizeof(T)), 8 * sizeof(T));
    } else {
      T v[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        DT<T>::store1(v + e, 0.f);
        if (e < left) v[e] = q[e];
      }
      __builtin_memcpy(&f, v, 8 * sizeof(T));
    }
    return f;
  };
  for (int k0 = wave * 32 * U; k0 < p.K; k0 += 8 * 32 * U) {
    LFrag<T> fw[U], fx[U][MI];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int left = p.K - (k0 + u * 32 + g * 8);
      fw[u] = get(w + k0 + u * 32, n < p.N ? left : 0);
#pragma unroll
      for (int i = 0; i < MI; ++i) fx[u][i] = get(x + (int64_t)i * 16 * p.lda + k0 + u * 32, i * 16 + c < p.M ? left : 0);
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
  const int64_t chunks = pitch / K::VEC;
  for (int64_t x = (int64_t)blockIdx.x * 256 + threadIdx.x; x < rows * chunks; x += (int64_t)gridDim.x * 256) {
    const int64_t row = x / chunks;
    const int c = (int)(x - row * chunks) * K::VEC;
    float v[K::VEC];
    K::load(src + row * ld + c, n - c, v);
    K::store(dst + row * pitch + c, K::VEC, v);
  }
}

// -------------------------------------------------------------------------------------------------------------------------------- host
struct LinPick {
  int tile;                                // 256, 128 or 64 rows and columns to a block
  int splits, split_tiles;
};

// Tile and splits by an estimate in cycles, from what the kernel measured (bf16 / fp32, 14 shapes from 300 x 256 x 256 to 8192 x 4096 x 4096, every tile and
// 1 to 16 splits): a compute unit works a 64- / 128- / 256-row tile's 128 bytes of k off in 455 / 1214 / 3825 cycles (fp32: 1367 / 5500) where blocks share it, in no
// less than 624 / 1170 / 2930 (2100 / 5500) alone; a block costs 1500 / 3000 / 8000 besides, a launch 8700 / 13500 / 20400 (the larger tiles' first loads and last
// stores).  A split keeps four tiles of k, and adds its partial results' way through memory (2 KB a cycle) and a launch of 10000.  Within 10 % of the best
// choice on 37 of the 42 products.
static LinPick lin_pick(int M, int N, int K, int es) {
  static const struct { int tile; double shared[2], alone[2], block, launch; } kind[3] = {
      {64, {455, 1367}, {624, 2100}, 1500, 8700}, {128, {1214, 5500}, {1170, 5500}, 3000, 13500}, {256, {3825, 0}, {2930, 0}, 8000, 20400}};
  const int nk = (int)(((int64_t)K * es + 127) / 128), wide = es == 4;
  LinPick best{128, 1, nk};
  double least = 0;
  for (const auto& q : kind) {
    if (q.tile == 256 && wide) break;                                          // (fp32: 3 times the 64-row tiles' time)
    const int64_t tiles = (int64_t)((M + q.tile - 1) / q.tile) * ((N + q.tile - 1) / q.tile);
    for (int s = 1; s <= 16 && (s == 1 || (q.tile < 256 && nk / s >= 4)); ++s) {
      const int per = (nk + s - 1) / s;
      if ((nk + per - 1) / per != s) continue;                                 // (the same as a smaller split)
      // (lin_check has seen to it that one does)
      if (!grid_fits(tiles * s, q.tile == 256 ? 512 : 256) || (s > 1 && !grid_fits(((int64_t)M * ((N + 3) / 4) + 255) / 256, 256))) continue;
      const double busy = (double)((tiles * s + 255) / 256);
      const double work = per * (busy * q.shared[wide] > q.alone[wide] ? busy * q.shared[wide] : q.alone[wide]);
      const double cost = work + busy * q.block + q.launch + (s > 1 ? 10000 + (double)(s + 1) * M * N * 4 / 2000 : 0);
      if (least == 0 || cost < least) {
        least = cost;
        best = {q.tile, s, per};
      }
    }
  }
  return best;
}

static int64_t lin_round(int64_t bytes) { return (bytes + 255) / 256 * 256; }
static int lin_es(int dtype) { return dtype == MOY_F32 ? 4 : 2; }
// rows of n elements that the tiled kernel can take as they are: whole dwords
static bool lin_direct(const void* p, int64_t ld, int n, int es) {
  return reinterpret_cast<uintptr_t>(p) % 4 == 0 && ld * es % 4 == 0 && (int64_t)n * es % 4 == 0;
}
static int64_t lin_span(int64_t rows, int64_t ld, int64_t n, int es) { return ((rows - 1) * ld + n) * es; }
static int64_t lin_pitch(int n, int es) { return ((int64_t)n * es + 15) / 16 * 16 / es; }

// Few rows go through lin_few_kernel, which asks for W in one wave of loads after another: up to 32 rows of up to 2048 elements, up to 16 of any length in fp32, whose tiled
// kernel pays four times as much for the rows that are not there (us, against the tiled kernel; 1, 16, 32 rows.  bf16: 256 -> 256 3.6 / 4.5, 2.9 / 4.6, 3.3 / 4.7;
// 1024 -> 4096 4.2 / 7.9, 4.4 / 8.0, 5.5 / 8.0; 2048 -> 4096 6.3 / 7.5, 6.4 / 8.1, 8.4 / 8.8; 4096 -> 1024 8.0 / 7.3, 9.5 / 8.4, 13.0 / 8.6; 4096 -> 4096 10.5 / 9.8, 9.9 / 10.6,
// 14.1 / 12.4; 8192 -> 8192 31.7 / 24.3, 31.9 / 24.9, 45.7 / 25.3.  fp32: 1024 -> 4096 6.1 / 11.5, 7.0 / 12.1, 9.4 / 13.2; 2048 -> 2048 8.7 / 12.0, 11.1 / 12.6, 15.5 / 13.5;
// 4096 -> 1024 14.8 / 12.2, 17.8 / 12.7, 26.9 / 13.2; 4096 -> 4096 19.3 / 25.6, 19.3 / 25.8, 28.1 / 26.1; 8192 -> 8192 55 / 80, 65 / 80, 102 / 81).
static bool lin_few(int M, int K, int es) { return M <= (K <= 2048 ? 32 : es == 4 ? 16 : 0); }

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
  constexpr int VEC = 16 / (int)sizeof(T);
  p.clamp = (ACOL ? p.M : p.K) % VEC != 0 || (BCOL ? p.N : p.K) % VEC != 0;
  const dim3 grid((unsigned)((int64_t)p.tiles_m * p.tiles_n * k.splits));
#define MOY_LIN(WM, WN, MI, NI, ST)                                                                                                     \
  {                                                                                                                                 \
    auto kern = lin_gemm_kernel<T, ACOL, BCOL, WM, WN, MI, NI, ST>;                                                                     \
    static std::atomic<uint64_t> ready{0};                                                                                              \
    const int rc = lds_opt_in(reinterpret_cast<const void*>(kern), ready);                                                              \
    if (rc != MOY_OK) return rc;                                                                                                    \
    hipLaunchKernelGGL(kern, grid, dim3(WM * WN * 64), ST * 128 * (WM * MI * 16 + WN * NI * 16), st, p);                               \
  }
  if (sizeof(T) == 2 && k.tile == 256) {
    if constexpr (sizeof(T) == 2) MOY_LIN(2, 4, 8, 4, 2)
  } else if (k.tile == 128) MOY_LIN(2, 2, 4, 4, 2)
  else MOY_LIN(2, 2, 2, 2, 3)
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
  const int64_t blocks = (rows * (pitch / Chunk<T>::VEC) + 255) / 256, most = 1 << 20;   // (blocks beyond that go round again)
  hipLaunchKernelGGL((lin_pad_kernel<T>), dim3((unsigned)(blocks < most ? blocks : most)), dim3(256), 0, st, static_cast<const T*>(src), ld, rows, n, static_cast<T*>(dst), pitch);
  return launch_status();
}

static int lin_check(const moy_linear_args* a, bool bwd) {
  if (!a || a->dtype < MOY_F32 || a->dtype > MOY_F16 || a->M <= 0 || a->N <= 0 || a->K <= 0) return MOY_EINVAL;
  if (a->act < MOY_ACT_NONE || a->act > MOY_ACT_SIGMOID || (a->b_dtype != MOY_F32 && a->b_dtype != a->dtype)) return MOY_EINVAL;
  const int d = a->dtype;
  if (!a->x || !a->w || !aligned_as(a->x, d) || !aligned_as(a->w, d) || (a->M > 1 && a->ldx < 0) || (a->N > 1 && a->ldw < 0)) return MOY_EINVAL;
  // rows up to 4 MiB long, and no further apart where the tiled kernel addresses them (by 32-bit offsets within a tile); lin_few_kernel takes any distance
  const bool few = !bwd && lin_few(a->M, a->K, lin_es(d));
  auto apart = [&](int64_t ld, int rows) { return !few && rows > 1 && ld > (1 << 22) / lin_es(d); };
  if ((int64_t)a->K * lin_es(d) > (1 << 22) || (int64_t)a->N * lin_es(d) > (1 << 22) || apart(a->ldx, a->M) || apart(a->ldw, a->N)) return MOY_ENOSYS;
  // row numbers a tile past the last one are still whole numbers of 32 bits, and each product has a grid that can be launched (in 128-row tiles, if in no others)
  auto fits = [](int64_t m, int64_t n) { return grid_fits((m + 127) / 128 * ((n + 127) / 128), 256); };
  if (a->M > 0x7fffffff - 512 || (!bwd && !fits(a->M, a->N)) || (bwd && ((a->dx && !fits(a->M, a->K)) || (a->dw && !fits(a->N, a->K))))) return MOY_ENOSYS;
  if (!bwd) {
    if (apart(a->ldy, a->M) || (a->r && apart(a->ldr, a->M))) return MOY_ENOSYS;
    if (!a->y || !aligned_as(a->y, d) || (a->M > 1 && a->ldy < a->N) || !aligned_as(a->b, a->b_dtype)) return MOY_EINVAL;
    if (!aligned_as(a->r, d) || (a->r && a->M > 1 && a->ldr < 0) || !aligned_as(a->z, d)) return MOY_EINVAL;
  } else {
    if (!a->dy || !aligned_as(a->dy, d) || (a->M > 1 && a->ldd < 0) || (!a->dx && !a->dw && !a->db)) return MOY_EINVAL;
    if ((a->act != MOY_ACT_NONE && !a->z) || !aligned_as(a->z, d) || !aligned_as(a->dx, d) || !aligned_as(a->dw, d) || !aligned_as(a->db, a->b_dtype)) return MOY_EINVAL;
    if (apart(a->ldd, a->M)) return MOY_ENOSYS;
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
  const bool few = !bwd && lin_few(a->M, a->K, es);                            // (takes any rows)
  p.pad_x = !few && (!bwd || a->dw) && !lin_direct(a->x, a->ldx, a->K, es);
  p.pad_w = !few && (!bwd || a->dx) && !lin_direct(a->w, a->ldw, a->K, es);
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
    if (!few) at += lin_part_bytes(a->M, a->N, a->K, es);
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
  p.a_bytes = lin_span(a->M, p.lda, plan.pad_x ? pitch : a->K, sizeof(T));
  p.b_bytes = lin_span(a->N, p.ldb, plan.pad_w ? pitch : a->K, sizeof(T));
  p.M = a->M; p.N = a->N; p.K = a->K;
  p.bias = a->b; p.bias_dtype = a->b_dtype; p.act = a->act;
  p.r = a->r; p.ldr = a->ldr; p.y = a->y; p.ldy = a->ldy; p.z = a->z; p.ldz = a->N;
  if (lin_few(a->M, a->K, sizeof(T))) {
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
    p.a_bytes = lin_span(a->M, ldz, plan.make_dz ? np : a->N, ES);
    p.b_bytes = lin_span(a->N, p.ldb, plan.pad_w ? kp : a->K, ES);
    p.M = a->M; p.N = a->K; p.K = a->N;
    p.y = a->dx; p.ldy = a->K;
    if ((rc = lin_gemm<T, false, true>(p, part, st)) != MOY_OK) return rc;
  }
  if (a->dw) {
    LinParams p{};
    p.a = dz; p.lda = ldz;
    p.b = plan.pad_x ? ws + plan.x : a->x;
    p.ldb = plan.pad_x ? kp : a->ldx;
    p.a_bytes = lin_span(a->M, ldz, plan.make_dz ? np : a->N, ES);
    p.b_bytes = lin_span(a->M, p.ldb, plan.pad_x ? kp : a->K, ES);
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
