// Attention with a learned relative position bias by buckets, forward and backward.
//
//   S_ij = scale q_i . k_j + table[lut[clamp(j - (i + start), -far, far) + far], h]     (log2 units here: scale and bias carry log2 e)
//   P = softmax_j S over the keys that count     O = P V          empty rows: O = 0, no gradient
//   dP = dO V^T    dS = P (dP - delta), delta_i = dO_i . O_i      dq = scale dS K    dK = scale dS^T Q    dV = P^T dO    dtable[b] = sum of dS in bucket b
//
// One pass over the keys with a running maximum and sum (fp32).  All products run on the matrix cores, in 16x16 tiles: 16-bit types take K = 32 at a time, fp32
// exact products of K = 4 at a time in the same register layout.  In 16-bit types the forward's P enters its product as two operands, its rounded value and
// what that leaves out: the backward takes dO . O for sum_j P_ij dP_ij, and what O missed of that would not cancel in dtable, where rows of dS add up
// to 0 (a quarter of the forward's time at 2 x 4096; without it dtable was up to 2.4 times, o 1.4 times as far off as one rounding).  P and dS of the
// backward are rounded to 16 bits once: nothing there adds up to 0, and dq, dk and dv are 2.4e-3 off in norm (bf16, 2 x 4096) where the rounding of an exact result alone makes
// 1.7e-3; both as two operands made it that, for 233 us of dQ instead of 206 and 281 of dK and dV instead of 215.  Who wants neither rounding computes in fp32.
// The products are laid out so that
// probabilities never leave registers: S^T = K Q^T puts a query in a lane's column and four consecutive keys in its accumulator, which is (keys permuted
// alike on both sides) the operand that O^T = V^T P^T takes.  V^T, K^T, Q^T, dO^T operands come out of row-major LDS tiles through the transposing LDS
// read (16-bit) or by single elements (fp32).  A row's maximum, sum, delta and position are one lane's scalars; only the maximum crosses lanes.
//
// Kernels: attn_fwd_kernel (a block takes 64 * NQ queries of one head, tiles of keys double-buffered in LDS); attn_split_kernel (few queries over a long cache:
// 16 (query, head of a shared group) rows to a block, the keys split over waves and blocks, partial results joined in split order); attn_dq_kernel (dQ,
// delta, sums of dtable); attn_dkv_kernel (dK, dV: a block owns keys and walks the queries of every head that shares them).  The two backward kernels
// compute S twice instead of adding dQ atomically: results do not depend on the order in which blocks run.
//
// Measured: 2 x 4096 causal, 16 heads of 64, bf16: forward 152 us, dQ 208, dK and dV 217 (450, 495 and 635 TFLOP/s).  By its counters the forward is bound by the vector units: they
// are busy 73 % of the time (320 instructions of a wave for 64 keys x 32 queries, 32 of them exponentials at four times the price), the matrix cores 35 % (48 instructions), at 2.7
// waves to a SIMD.  dQ and dK / dV keep the vector units busy for 51 and 52 %, the matrix cores for 24 and 31 %, the LDS for 21 and 25 %: their registers leave 1.9 waves to a SIMD,
// each of which waits a third of its time for data, with too little beside it to fill in.  Heads of 128 take 277, 394 and 523, heads of 96 as much (they are padded to 128), at 16
// queries or keys to a wave.  fp32, 4 x 1024 causal, 16 heads of 64: 109, 171, 185.  16 x 300 with a mask by query, 8 heads of 32, fp16: 17, 26, 19: five tiles to a block, latency.
// One query for each of 32 caches of up to 16384 keys, 16 heads over 4 key heads of 64: 78 us and 4.8 to join, 5.1 TB/s over the keys that count; full caches of 16384, heads of 64
// in fp32 or of 128 in bf16 193 and 197 (5.5), of 128 in fp32 423 (5.1, with 20 bytes of a lane spilled).  The backward does not split the keys: 16 queries, 4096 keys, 8 heads of 64 are eight blocks and 86 us of dQ.
#include "common.hpp"

namespace moy {

constexpr float LOG2E = 1.4426950408889634f;

struct AttnParams {
  const void *q, *k, *v;
  int64_t q_sb, q_sl, q_sh, k_sb, k_sl, k_sh, v_sb, v_sl, v_sh;
  int B, H, Hk, Lq, Lk, D;
  const void* table; const uint8_t* lut; int nb, far;
  const int32_t* k_len; int q_from_end, q_start, causal;
  const uint8_t* mask; int64_t m_sb, m_sh, m_sq;
  float scale, scale2;                     // scale2 = scale log2 e
  void* o; float* lse;                     // lse fp32 [B, H, Lq], log2 units; -inf: an empty row
  void* rest;                              // 16-bit types: what the rounding of o left out (o + rest: 16 bits or more of mantissa), for delta
  const void* dout; int64_t g_sb, g_sl, g_sh;
  void *dq, *dk, *dv;
  float* delta;                            // backward: fp32 [B, H, Lq]
  float* part;                             // backward: fp32 [H][B * query tiles][nb] sums of dS; split forward: partial results
  int tiles, splits, split_keys;           // row tiles of a (batch, head); key splits of the split forward and their length
};

// ---- matrix operands: 8 elements of one row / column for a lane (l % 16 = row or column, l / 16 = which eight of 32)
template <typename T>
struct Frag {
  u32x4 w;
};
template <>
struct Frag<float> {
  f32x4 lo, hi;
};
__device__ __forceinline__ f32x4 attn_mma(f32x4 acc, const Frag<bf16_t>& a, const Frag<bf16_t>& b) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a.w), __builtin_bit_cast(bf16x8, b.w), acc, 0, 0, 0);
}
__device__ __forceinline__ f32x4 attn_mma(f32x4 acc, const Frag<f16_t>& a, const Frag<f16_t>& b) {
  return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a.w), __builtin_bit_cast(f16x8, b.w), acc, 0, 0, 0);
}
__device__ __forceinline__ f32x4 attn_mma(f32x4 acc, const Frag<float>& a, const Frag<float>& b) {
  acc = __builtin_amdgcn_mfma_f32_16x16x4f32(a.lo.x, b.lo.x, acc, 0, 0, 0);
  acc = __builtin_amdgcn_mfma_f32_16x16x4f32(a.lo.y, b.lo.y, acc, 0, 0, 0);
  acc = __builtin_amdgcn_mfma_f32_16x16x4f32(a.lo.z, b.lo.z, acc, 0, 0, 0);
  acc = __builtin_amdgcn_mfma_f32_16x16x4f32(a.lo.w, b.lo.w, acc, 0, 0, 0);
  acc = __builtin_amdgcn_mfma_f32_16x16x4f32(a.hi.x, b.hi.x, acc, 0, 0, 0);
  acc = __builtin_amdgcn_mfma_f32_16x16x4f32(a.hi.y, b.hi.y, acc, 0, 0, 0);
  acc = __builtin_amdgcn_mfma_f32_16x16x4f32(a.hi.z, b.hi.z, acc, 0, 0, 0);
  acc = __builtin_amdgcn_mfma_f32_16x16x4f32(a.hi.w, b.hi.w, acc, 0, 0, 0);
  return acc;
}
// (DT<f16_t>::pack2 pins its operands in registers, which costs this file's loops a wave of occupancy)
template <typename T>
__device__ __forceinline__ uint32_t pack_as(float lo, float hi) {
  typedef _Float16 h2 __attribute__((ext_vector_type(2)));
  if constexpr (DT<T>::code == MOY_F16) return __builtin_bit_cast(uint32_t, __builtin_convertvector(f32x2_{lo, hi}, h2));
  else return pack_bf2(lo, hi);
}
// two accumulators (rows 4 q .. 4 q + 3 of two 16-row tiles) -> the operand whose lane holds those eight
template <typename T>
__device__ __forceinline__ Frag<T> frag_of(const f32x4& a, const f32x4& b) {
  if constexpr (sizeof(T) == 4) return Frag<T>{a, b};
  else return Frag<T>{u32x4{pack_as<T>(a.x, a.y), pack_as<T>(a.z, a.w), pack_as<T>(b.x, b.y), pack_as<T>(b.z, b.w)}};
}
// what rounding to that operand left out, as another one
template <typename T>
__device__ __forceinline__ Frag<T> frag_rest(const f32x4& a, const f32x4& b, const Frag<T>& f) {
  static_assert(sizeof(T) == 2, "nothing is rounded in fp32");
  const uint32_t w[4] = {f.w.x, f.w.y, f.w.z, f.w.w};
  return Frag<T>{u32x4{pack_as<T>(a.x - DT<T>::lo(w[0]), a.y - DT<T>::hi(w[0])), pack_as<T>(a.z - DT<T>::lo(w[1]), a.w - DT<T>::hi(w[1])),
                       pack_as<T>(b.x - DT<T>::lo(w[2]), b.y - DT<T>::hi(w[2])), pack_as<T>(b.z - DT<T>::lo(w[3]), b.w - DT<T>::hi(w[3]))}};
}
// eight consecutive elements of a row, in memory or LDS (16-byte aligned)
template <typename T>
__device__ __forceinline__ Frag<T> frag_row(const T* p) {
  if constexpr (sizeof(T) == 4) return Frag<T>{*reinterpret_cast<const f32x4*>(p), *reinterpret_cast<const f32x4*>(p + 4)};
  else return Frag<T>{*reinterpret_cast<const u32x4*>(p)};
}
template <typename T>
__device__ __forceinline__ Frag<T> frag_zero() {
  if constexpr (sizeof(T) == 4) return Frag<T>{f32x4{0.f, 0.f, 0.f, 0.f}, f32x4{0.f, 0.f, 0.f, 0.f}};
  else return Frag<T>{u32x4{0u, 0u, 0u, 0u}};
}
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) s16x4* lds_s16x4;
// the transposed operand of a row-major LDS tile: lane (c = l % 16, g = l / 16) gets column col0 + c of rows row0 + 4 g + 0..3 and row0 + 16 + 4 g + 0..3
// (the order in which frag_of lays down accumulators)
template <typename T, int PITCH>
__device__ __forceinline__ Frag<T> frag_cols(const T* tile, int row0, int col0, int lane) {
  if constexpr (sizeof(T) == 4) {
    const float* p = reinterpret_cast<const float*>(tile) + (row0 + 4 * (lane >> 4)) * PITCH + col0 + (lane & 15);
    return Frag<T>{f32x4{p[0], p[PITCH], p[2 * PITCH], p[3 * PITCH]}, f32x4{p[16 * PITCH], p[17 * PITCH], p[18 * PITCH], p[19 * PITCH]}};
  } else {
    const T* p = tile + (row0 + 4 * (lane >> 4) + ((lane >> 2) & 3)) * PITCH + col0 + 4 * (lane & 3);
    const s16x4 a = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4)(const_cast<T*>(p)));
    const s16x4 b = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4)(const_cast<T*>(p + 16 * PITCH)));
    const u32x2 x = __builtin_bit_cast(u32x2, a), y = __builtin_bit_cast(u32x2, b);
    return Frag<T>{u32x4{x.x, x.y, y.x, y.y}};
  }
}
// across the four lanes (l, l ^ 16, l ^ 32, l ^ 48) that share a column
__device__ __forceinline__ float cols_max(float v) {
  typedef uint32_t pair __attribute__((ext_vector_type(2)));
  uint32_t u = __builtin_bit_cast(uint32_t, v);
  pair r = __builtin_bit_cast(pair, __builtin_amdgcn_permlane16_swap(u, u, false, false));
  uint32_t x = r.x, y = r.y;
  v = fmaxf(__builtin_bit_cast(float, x), __builtin_bit_cast(float, y));
  u = __builtin_bit_cast(uint32_t, v);
  r = __builtin_bit_cast(pair, __builtin_amdgcn_permlane32_swap(u, u, false, false));
  x = r.x;
  y = r.y;
  return fmaxf(__builtin_bit_cast(float, x), __builtin_bit_cast(float, y));
}
__device__ __forceinline__ float cols_sum(float v) {
  v += __shfl_xor(v, 16);
  return v + __shfl_xor(v, 32);
}

// o = v rounded, and what the rounding left out
template <typename T>
__device__ __forceinline__ void store_o(T* o, T* rest, int64_t at, f32x4 v) {
  DT<T>::store4(o + at, v);
  if constexpr (sizeof(T) == 2) {
    if (rest) {
      const uint32_t a = DT<T>::pack2(v.x, v.y), b = DT<T>::pack2(v.z, v.w);
      DT<T>::store4(rest + at, f32x4{v.x - DT<T>::lo(a), v.y - DT<T>::hi(a), v.z - DT<T>::lo(b), v.w - DT<T>::hi(b)});
    }
  }
}
template <typename T>
__device__ __forceinline__ void store_o1(T* o, T* rest, int64_t at, float v) {
  DT<T>::store1(o + at, v);
  if constexpr (sizeof(T) == 2) {
    if (rest) DT<T>::store1(rest + at, v - DT<T>::lo(DT<T>::pack2(v, v)));
  }
}

// ---- a [ROWS][DP] tile of a strided tensor: 256 threads take 16-byte chunks, columns past D and rows that do not count are zeros
template <typename T, int DP, int ROWS, int THREADS>
struct Tile {
  static constexpr int VEC = DT<T>::KPB, CH = DP / VEC, N = ROWS * CH / THREADS, PITCH = DP + 32 / (int)sizeof(T);   // 32 bytes of padding: row and transposed reads without bank conflicts (16 bytes: 38 % of the LDS cycles were conflicts)
  static_assert(N * THREADS == ROWS * CH, "whole chunks");
  static constexpr int BYTES = ROWS * PITCH * (int)sizeof(T);
  u32x4 r[N];
  __device__ __forceinline__ void load(const T* base, int64_t ld, int row0, int rows, int D, const uint8_t* hide, int tid) {
    if (row0 + ROWS <= rows && D == DP && !hide) {
#pragma unroll
      for (int n = 0; n < N; ++n) {
        const int c = tid + n * THREADS;
        r[n] = *reinterpret_cast<const u32x4*>(base + (int64_t)(row0 + c / CH) * ld + c % CH * VEC);
      }
      return;
    }
#pragma unroll
    for (int n = 0; n < N; ++n) {
      const int c = tid + n * THREADS, row = row0 + c / CH, col = c % CH * VEC;
      const bool in = row < rows && col < D && !(hide && hide[row]);
      r[n] = in ? *reinterpret_cast<const u32x4*>(base + (int64_t)row * ld + col) : u32x4{0u, 0u, 0u, 0u};
    }
  }
  __device__ __forceinline__ void store(T* lds, int tid) const {
#pragma unroll
    for (int n = 0; n < N; ++n) {
      const int c = tid + n * THREADS;
      *reinterpret_cast<u32x4*>(lds + (c / CH) * PITCH + c % CH * VEC) = r[n];
    }
  }
};

// XCD-aware order: the blocks of one XCD take consecutive tiles, so that the tiles of a head share its keys in one L2
__device__ __forceinline__ int xcd_order(int bid, int nb) {
  const int qd = nb >> 3, rm = nb & 7, x = bid & 7;
  return (x < rm ? x * (qd + 1) : rm * (qd + 1) + (x - rm) * qd) + (bid >> 3);
}

// Which (batch, head) and tile a block takes.  Without a causal mask a head's tiles follow one another.  With one the tiles differ in length: the long
// ones (tile p.tiles - 1 first) of the heads of an XCD come first, the short ones fill in behind them.
__device__ __forceinline__ void tile_order(const AttnParams& p, int id, int heads, int* head, int* tile) {
  if (p.causal && heads % 8 == 0) {
    const int per = heads / 8, x = id / (per * p.tiles), y = id - x * per * p.tiles;
    *tile = p.tiles - 1 - y / per;
    *head = x * per + y % per;
  } else {
    *head = id / p.tiles;
    *tile = p.tiles - 1 - (id - *head * p.tiles);
  }
}

// What a (batch, head) attends over.
struct Span {
  int klen, start;                         // keys that count; position of query 0
  const uint8_t* mask; int64_t m_sq;       // mask + query * m_sq + key: not 0 = hidden
  const uint8_t* hide;                     // the same row for every query: hidden keys' rows are not read at all
};
__device__ __forceinline__ Span span_of(const AttnParams& p, int b, int h) {
  Span s;
  s.klen = p.Lk;
  if (p.k_len) s.klen = min(max(p.k_len[b], 0), p.Lk);
  s.start = p.q_from_end ? s.klen - p.Lq : p.q_start;
  s.mask = p.mask ? p.mask + b * p.m_sb + h * p.m_sh : nullptr;
  s.m_sq = p.m_sq;
  s.hide = p.mask && p.m_sq == 0 ? s.mask : nullptr;
  return s;
}

// The bias of one head by clamped distance, four constant entries beyond each end (so that four neighbours are one read wherever they lie):
// entry e stands for distance e - 4 - far.
template <typename T>
__device__ __forceinline__ void load_bias(const AttnParams& p, int h, float* bias, int threads) {
  for (int e = threadIdx.x; e < 2 * p.far + 9; e += threads) {
    const int at = min(max(e - 4, 0), 2 * p.far);
    bias[e] = DT<T>::load1(static_cast<const T*>(p.table) + (int64_t)min((int)p.lut[at], p.nb - 1) * p.H + h) * LOG2E;
  }
}
// entry of the first of four neighbours at distances d .. d + 3
__device__ __forceinline__ int bias_at(int d, int far) { return min(max(d, -far - 4), far + 1) + far + 4; }

__device__ __forceinline__ f32x4 bias4(const float* p) { return f32x4{p[0], p[1], p[2], p[3]}; }

// does the tile of keys [j0, j0 + nk) against positions [p0, p1] lie wholly beyond one end (its bias is one number)?  -1 / 1: before / after, 0: no
__device__ __forceinline__ int beyond(int j0, int nk, int p0, int p1, int far) { return j0 + nk - 1 - p0 <= -far ? -1 : j0 - p1 >= far ? 1 : 0; }

// four mask bytes of keys j .. j + 3 (bytes past the last key: hidden)
__device__ __forceinline__ uint32_t mask4(const uint8_t* m, int j, int lk) {
  uint32_t w = 0x01010101u;
  if (j + 4 <= lk) {
    __builtin_memcpy(&w, m + j, 4);
  } else {
#pragma unroll
    for (int e = 0; e < 4; ++e)
      if (j + e < lk) w = (w & ~(0xffu << (8 * e))) | ((uint32_t)m[j + e] << (8 * e));
  }
  return w;
}

// A [ROWS queries][COLS keys] tile of mask bytes as bits in LDS (1: hidden), loaded ahead like the tiles it goes with: 256 threads take 8 or 16 bytes each.
// Queries past the last repeat the last one's row, and bits past the last key are anything: neither is looked at.
template <int ROWS, int COLS>
struct MaskTile {
  static constexpr int EACH = ROWS * COLS / 256, CB = EACH < 16 ? EACH : 16, N = EACH / CB, CH = COLS / CB, WORDS = COLS / 32, BYTES = ROWS * COLS / 8;
  static_assert(CB >= 8 && N * CB == EACH, "whole chunks");
  typedef uint32_t chunk __attribute__((ext_vector_type(CB / 4)));
  chunk r[N];
  __device__ __forceinline__ void load(const uint8_t* m, int64_t ld, int row0, int rows, int col0, int cols, int tid) {
#pragma unroll
    for (int n = 0; n < N; ++n) {
      const int c = tid + n * 256, col = col0 + c % CH * CB;
      const uint8_t* row = m + (int64_t)min(row0 + c / CH, rows - 1) * ld;
      if (cols >= CB) {
        __builtin_memcpy(&r[n], row + min(col, cols - CB), CB);                // the last chunk ends with the row, and is shifted below
      } else {
#pragma unroll
        for (int w = 0; w < CB / 4; ++w) {
          uint32_t v = 0u;
#pragma unroll
          for (int e = 0; e < 4; ++e)
            if (col + 4 * w + e < cols) v |= (uint32_t)row[col + 4 * w + e] << (8 * e);
          r[n][w] = v;
        }
      }
    }
  }
  __device__ __forceinline__ void store(uint32_t* lds, int col0, int cols, int tid) const {
#pragma unroll
    for (int n = 0; n < N; ++n) {
      const int c = tid + n * 256, col = col0 + c % CH * CB;
      uint32_t bits = 0u;
#pragma unroll
      for (int w = 0; w < CB / 4; ++w) {
        const uint32_t v = r[n][w], any = ((((v & 0x7f7f7f7fu) + 0x7f7f7f7fu) | v) >> 7) & 0x01010101u;   // a byte that is not 0: its lowest bit
        bits |= (any * 0x01020408u >> 24 & 15u) << (4 * w);                    // the four gathered (no two products meet)
      }
      const int past = cols >= CB ? min(col - min(col, cols - CB), 31) : 0;
      if constexpr (CB == 16) reinterpret_cast<uint16_t*>(lds)[c] = (uint16_t)(bits >> past);
      else reinterpret_cast<uint8_t*>(lds)[c] = (uint8_t)(bits >> past);
    }
  }
};
// the bits of 32 keys from the one `left` short of the end on: those that do not count
__device__ __forceinline__ uint32_t past_bits(int left) { return left >= 32 ? 0u : ~0u << max(left, 0); }
// all ones where bit b is set (in assembly: the compiler makes a comparison and a selection of it, with a wait between them)
__device__ __forceinline__ uint32_t bit_mask(uint32_t w, int b) {
  uint32_t all;
  asm("v_bfe_i32 %0, %1, %2, 1" : "=v"(all) : "v"(w), "n"(b));
  return all;
}
__device__ __forceinline__ float pick(uint32_t all, float set, float v) {
  return __builtin_bit_cast(float, (__builtin_bit_cast(uint32_t, set) & all) | (__builtin_bit_cast(uint32_t, v) & ~all));
}

// fp16 holds a probability with all its bits only from 2^-14 on, and rows of some ten thousand keys are below that: where P is an operand on its own (dV), it is carried
// 2^15 times as large (at most 32768; in the exponent, the row's statistics and the result's scale, which costs nothing).
template <typename T>
constexpr float P_UP = DT<T>::code == MOY_F16 ? 32768.f : 1.f;
template <typename T>
constexpr float P_UP_LOG2 = DT<T>::code == MOY_F16 ? 15.f : 0.f;

// keys (backward of dK, dV: queries) of an LDS tile
template <typename T, int DP>
constexpr int attn_bk() { return sizeof(T) * DP <= 128 ? 64 : 32; }

// ------------------------------------------------------------------------------------------------------------------------------ forward
template <typename T, int DP, int NQ, int BK, bool MASK>
__global__ __launch_bounds__(256, 2) void attn_fwd_kernel(const AttnParams p) {
  constexpr int KP = DP / 32, DT16 = DP / 16, NKT = BK / 16, BQ = 64 * NQ;
  constexpr bool FINE = sizeof(T) == 2;                                        // P in two operands
  using TL = Tile<T, DP, BK, 256>;
  extern __shared__ __attribute__((aligned(16))) unsigned char smem[];
  T* kt_ = reinterpret_cast<T*>(smem);
  T* vt_ = reinterpret_cast<T*>(smem + 2 * TL::BYTES);
  using ML = MaskTile<BQ, BK>;
  uint32_t* mt_ = reinterpret_cast<uint32_t*>(smem + 4 * TL::BYTES);
  float* bias = reinterpret_cast<float*>(smem + 4 * TL::BYTES + 2 * ML::BYTES);
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), c = lane & 15, g = lane >> 4;
  const int id = xcd_order(blockIdx.x, gridDim.x);
  int bh, qt;
  tile_order(p, id, p.B * p.H, &bh, &qt);
  const int b = bh / p.H, h = bh - b * p.H, hk = h / (p.H / p.Hk);
  const Span sp = span_of(p, b, h);
  const T* kb = static_cast<const T*>(p.k) + b * p.k_sb + hk * p.k_sh;
  const T* vb = static_cast<const T*>(p.v) + b * p.v_sb + hk * p.v_sh;
  const int q0 = qt * BQ + wave * 16 * NQ;                                      // the wave's first query
  const int last = min(qt * BQ + BQ, p.Lq) - 1 + sp.start;                      // position of the block's last query
  const int kend = p.causal ? min(sp.klen, last + 1) : sp.klen;                // (no query of the block sees a key from here on: not read)
  const int nt = kend > 0 ? (kend + BK - 1) / BK : 0;

  Frag<T> qf[NQ][KP];
#pragma unroll
  for (int n = 0; n < NQ; ++n) {
    const int i = q0 + n * 16 + c;
    const T* qp = static_cast<const T*>(p.q) + b * p.q_sb + (int64_t)i * p.q_sl + h * p.q_sh + g * 8;
#pragma unroll
    for (int kp = 0; kp < KP; ++kp) qf[n][kp] = i < p.Lq && kp * 32 + g * 8 < p.D ? frag_row(qp + kp * 32) : frag_zero<T>();
  }
  f32x4 o[DT16][NQ];
  float m[NQ], l[NQ];
#pragma unroll
  for (int n = 0; n < NQ; ++n) {
    m[n] = -INFINITY;
    l[n] = 0.f;
#pragma unroll
    for (int d = 0; d < DT16; ++d) o[d][n] = f32x4{0.f, 0.f, 0.f, 0.f};
  }
  TL kr, vr;
  ML mr;
  if (nt > 0) {
    kr.load(kb, p.k_sl, 0, kend, p.D, MASK ? sp.hide : nullptr, tid);
    vr.load(vb, p.v_sl, 0, kend, p.D, MASK ? sp.hide : nullptr, tid);
    if constexpr (MASK) mr.load(sp.mask, sp.m_sq, qt * BQ, p.Lq, 0, p.Lk, tid);
    if (p.table) load_bias<T>(p, h, bias, 256);
    kr.store(kt_, tid);
    vr.store(vt_, tid);
    if constexpr (MASK) mr.store(mt_, 0, p.Lk, tid);
  }
  __syncthreads();
  for (int t = 0; t < nt; ++t) {
    const T* ks = kt_ + (t & 1) * (TL::BYTES / (int)sizeof(T));
    const T* vs = vt_ + (t & 1) * (TL::BYTES / (int)sizeof(T));
    const uint32_t* ms = mt_ + (t & 1) * (ML::BYTES / 4);
    const int j0 = t * BK;
    if (t + 1 < nt) {
      kr.load(kb, p.k_sl, j0 + BK, kend, p.D, MASK ? sp.hide : nullptr, tid);
      vr.load(vb, p.v_sl, j0 + BK, kend, p.D, MASK ? sp.hide : nullptr, tid);
      if constexpr (MASK) mr.load(sp.mask, sp.m_sq, qt * BQ, p.Lq, j0 + BK, p.Lk, tid);
    }
    f32x4 s[NKT][NQ];
#pragma unroll
    for (int kt = 0; kt < NKT; ++kt) {
#pragma unroll
      for (int n = 0; n < NQ; ++n) s[kt][n] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int kp = 0; kp < KP; ++kp) {
        const Frag<T> a = frag_row(ks + (kt * 16 + c) * TL::PITCH + kp * 32 + g * 8);
#pragma unroll
        for (int n = 0; n < NQ; ++n) s[kt][n] = attn_mma(s[kt][n], a, qf[n][kp]);
      }
    }
    const int p0 = q0 + sp.start, p1 = p0 + 16 * NQ - 1;                        // positions of the wave's queries
    const int far = p.table ? beyond(j0, BK, p0, p1, p.far) : -1;
    const bool cut = MASK || j0 + BK > sp.klen || (p.causal && j0 + BK - 1 > p0);
    Frag<T> pf[BK / 32][NQ], pr[FINE ? BK / 32 : 1][NQ];
    // One bias for the whole tile and every key counts: scale and bias wait for the exponential (scale >= 0: the largest product is the largest score).
    const bool plain = far && !cut;
    const float fixed = p.table && far ? bias[far < 0 ? 0 : 2 * p.far + 8] : 0.f;
    if (!plain) {
#pragma unroll
      for (int n = 0; n < NQ; ++n) {
        const int pos = q0 + n * 16 + c + sp.start;
        if (far) {
#pragma unroll
          for (int kt = 0; kt < NKT; ++kt) s[kt][n] = s[kt][n] * p.scale2 + fixed;
        } else {
          f32x4 w[NKT];
#pragma unroll
          for (int kt = 0; kt < NKT; ++kt) w[kt] = bias4(bias + bias_at(j0 + kt * 16 + 4 * g - pos, p.far));
#pragma unroll
          for (int kt = 0; kt < NKT; ++kt) s[kt][n] = s[kt][n] * p.scale2 + w[kt];
        }
        if (cut) {
          const int end = p.causal ? min(sp.klen, pos + 1) : sp.klen;
#pragma unroll
          for (int kc = 0; kc < BK / 32; ++kc) {
            uint32_t off = past_bits(end - j0 - kc * 32);
            if constexpr (MASK) off |= ms[(wave * 16 * NQ + n * 16 + c) * ML::WORDS + kc];
            off >>= 4 * g;
#pragma unroll
            for (int kt = 0; kt < 2; ++kt)
#pragma unroll
              for (int e = 0; e < 4; ++e) s[2 * kc + kt][n][e] = pick(bit_mask(off, kt * 16 + e), -INFINITY, s[2 * kc + kt][n][e]);
          }
        }
      }
    }
    const float mul = plain ? p.scale2 : 1.f, plus = plain ? fixed : 0.f;
    float top[NQ];
    bool grown = false;
#pragma unroll
    for (int n = 0; n < NQ; ++n) {
      top[n] = -INFINITY;
#pragma unroll
      for (int kt = 0; kt < NKT; ++kt)
#pragma unroll
        for (int e = 0; e < 4; ++e) top[n] = fmaxf(top[n], s[kt][n][e]);
      top[n] = cols_max(__builtin_fmaf(top[n], mul, plus));
      grown |= top[n] > m[n] + 8.f;
    }
    // The reference of the exponentials follows the maximum only where that has grown by more than 2^8: weights stay below 256, which costs nothing of
    // their precision, and the sums are seldom scaled.  (m = -inf at first: then the reference is the maximum, and a lone key weighs exactly 1.)
    if (__any(grown)) {
#pragma unroll
      for (int n = 0; n < NQ; ++n) {
        const float next = top[n] > m[n] + 8.f ? top[n] : m[n], f = next == m[n] ? 1.f : __builtin_amdgcn_exp2f(m[n] - next);
        l[n] *= f;
#pragma unroll
        for (int d = 0; d < DT16; ++d) o[d][n] *= f;
        m[n] = next;
      }
    }
#pragma unroll
    for (int n = 0; n < NQ; ++n) {
      const float ref = plus - (m[n] == -INFINITY ? 0.f : m[n]);                // nothing counted yet: exp2(-inf) below, not NaN
      f32x4 sum = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int kt = 0; kt < NKT; ++kt)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          s[kt][n][e] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[kt][n][e], mul, ref));
          sum[e] += s[kt][n][e];
        }
      l[n] += (sum.x + sum.y) + (sum.z + sum.w);
#pragma unroll
      for (int kc = 0; kc < BK / 32; ++kc) {
        pf[kc][n] = frag_of<T>(s[2 * kc][n], s[2 * kc + 1][n]);
        if constexpr (FINE) pr[kc][n] = frag_rest<T>(s[2 * kc][n], s[2 * kc + 1][n], pf[kc][n]);
      }
    }
#pragma unroll
    for (int d = 0; d < DT16; ++d)
#pragma unroll
      for (int kc = 0; kc < BK / 32; ++kc) {
        const Frag<T> a = frag_cols<T, TL::PITCH>(vs, kc * 32, d * 16, lane);
#pragma unroll
        for (int n = 0; n < NQ; ++n) {
          o[d][n] = attn_mma(o[d][n], a, pf[kc][n]);
          if constexpr (FINE) o[d][n] = attn_mma(o[d][n], a, pr[kc][n]);
        }
      }
    if (t + 1 < nt) {
      kr.store(kt_ + ((t + 1) & 1) * (TL::BYTES / (int)sizeof(T)), tid);
      vr.store(vt_ + ((t + 1) & 1) * (TL::BYTES / (int)sizeof(T)), tid);
      if constexpr (MASK) mr.store(mt_ + ((t + 1) & 1) * (ML::BYTES / 4), j0 + BK, p.Lk, tid);
    }
    __syncthreads();
  }
#pragma unroll
  for (int n = 0; n < NQ; ++n) {
    const int i = q0 + n * 16 + c;
    const float sum = cols_sum(l[n]);
    const float inv = sum == 0.f ? 0.f : 1.f / sum;
    if (i >= p.Lq) continue;
    if (p.lse && g == 0) p.lse[((int64_t)b * p.H + h) * p.Lq + i] = sum == 0.f ? -INFINITY : m[n] + __builtin_amdgcn_logf(sum);
    const int64_t at = (((int64_t)b * p.Lq + i) * p.H + h) * p.D + g * 4;
#pragma unroll
    for (int d = 0; d < DT16; ++d)
      if (d * 16 + g * 4 < p.D) store_o(static_cast<T*>(p.o), static_cast<T*>(p.rest), at + d * 16, o[d][n] * inv);
  }
}

// -------------------------------------------------------------------------------------------------------- few queries over many keys
// Rows are (query, head of the group that shares a key head): 16 to a block, so that the keys are read once for all of them.  A block takes one split of the
// keys, its four waves every fourth 32-key tile of it, each with a running maximum of its own: K comes from memory in operand order, V by way of
// the wave's own LDS tile; the waves are joined in LDS, the splits by attn_join_kernel.
template <typename T, int DP>
__global__ __launch_bounds__(256, 2) void attn_split_kernel(const AttnParams p) {
  constexpr int KP = DP / 32, DT16 = DP / 16;
  using TL = Tile<T, DP, 32, 64>;
  constexpr int VBYTES = 4 * TL::BYTES, OBYTES = 4 * 16 * (DP + 1) * 4;
  constexpr int BYTES = VBYTES > OBYTES ? VBYTES : OBYTES;
  __shared__ __attribute__((aligned(16))) unsigned char smem[BYTES];
  __shared__ float ml[4][16][2];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), c = lane & 15, g = lane >> 4;
  T* vs = reinterpret_cast<T*>(smem + wave * TL::BYTES);
  int id = blockIdx.x;
  const int turn = id % p.splits;
  id /= p.splits;
  const int split = (turn + id) % p.splits;                                    // (a block's number modulo 8 is its XCD: each takes early and late splits alike, since short sequences have no late ones)
  const int rt = id % p.tiles, bh = id / p.tiles, b = bh / p.Hk, hk = bh - b * p.Hk;
  const int share = p.H / p.Hk, rows = p.Lq * share, row = rt * 16 + c, i = row / share, h = hk * share + row - i * share;
  const bool live = row < rows;
  const Span sp = span_of(p, b, live ? h : hk * share);
  const int pos = i + sp.start;
  const T* kb = static_cast<const T*>(p.k) + b * p.k_sb + hk * p.k_sh;
  const T* vb = static_cast<const T*>(p.v) + b * p.v_sb + hk * p.v_sh;
  const int first = rt * 16 / share + sp.start, last = min((rt * 16 + 15) / share, p.Lq - 1) + sp.start;    // positions of the block's rows
  const int k0 = split * p.split_keys, kall = p.causal ? min(sp.klen, last + 1) : sp.klen, k1 = min(kall, k0 + p.split_keys);
  const int end = p.causal ? min(sp.klen, pos + 1) : sp.klen;
  const uint8_t* hide = sp.hide && p.m_sh == 0 ? sp.hide : nullptr;            // (a mask that differs by head hides rows of no key for all of them)
  float edge[2] = {0.f, 0.f};                                                  // the bias beyond either end
  if (p.table && live) {
#pragma unroll
    for (int s = 0; s < 2; ++s)
      edge[s] = DT<T>::load1(static_cast<const T*>(p.table) + (int64_t)min((int)p.lut[s * 2 * p.far], p.nb - 1) * p.H + h) * LOG2E;
  }
  Frag<T> qf[KP];
  const T* qp = static_cast<const T*>(p.q) + b * p.q_sb + (int64_t)i * p.q_sl + h * p.q_sh + g * 8;
#pragma unroll
  for (int kp = 0; kp < KP; ++kp) qf[kp] = live && kp * 32 + g * 8 < p.D ? frag_row(qp + kp * 32) : frag_zero<T>();
  f32x4 o[DT16];
#pragma unroll
  for (int d = 0; d < DT16; ++d) o[d] = f32x4{0.f, 0.f, 0.f, 0.f};
  float m = -INFINITY, l = 0.f;
  Frag<T> kf[2][KP];
  TL vr;
  auto load = [&](int j0) {
#pragma unroll
    for (int kt = 0; kt < 2; ++kt) {
      const int j = j0 + kt * 16 + c;
      const bool in = j < kall && !(hide && hide[j]);
      const T* kp_ = kb + (int64_t)j * p.k_sl + g * 8;
#pragma unroll
      for (int kp = 0; kp < KP; ++kp) kf[kt][kp] = in && kp * 32 + g * 8 < p.D ? frag_row(kp_ + kp * 32) : frag_zero<T>();
    }
    vr.load(vb, p.v_sl, j0, kall, p.D, hide, lane);
  };
  int j0 = k0 + wave * 32;
  if (j0 < k1) load(j0);
  for (; j0 < k1; j0 += 128) {
    f32x4 s[2];
#pragma unroll
    for (int kt = 0; kt < 2; ++kt) {
      s[kt] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int kp = 0; kp < KP; ++kp) s[kt] = attn_mma(s[kt], kf[kt][kp], qf[kp]);
    }
    vr.store(vs, lane);
    if (j0 + 128 < k1) load(j0 + 128);
    const int far = p.table ? beyond(j0, 32, first, last, p.far) : -1;
#pragma unroll
    for (int kt = 0; kt < 2; ++kt) {
      const int j = j0 + kt * 16 + 4 * g;
      const uint32_t w = sp.mask && live ? mask4(sp.mask + (int64_t)i * sp.m_sq, j, p.Lk) : 0u;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        float add = far < 0 ? edge[0] : edge[1];
        if (!far && live) {
          const int at = min(max(j + e - pos, -p.far), p.far) + p.far;
          add = DT<T>::load1(static_cast<const T*>(p.table) + (int64_t)min((int)p.lut[at], p.nb - 1) * p.H + h) * LOG2E;
        }
        const float x = s[kt][e] * p.scale2 + add;
        s[kt][e] = j + e >= end || ((w >> (8 * e)) & 0xffu) ? -INFINITY : x;
      }
    }
    float top = m;
#pragma unroll
    for (int kt = 0; kt < 2; ++kt)
#pragma unroll
      for (int e = 0; e < 4; ++e) top = fmaxf(top, s[kt][e]);
    top = cols_max(top);
    if (__any(top != m)) {
      const float f = top == m ? 1.f : __builtin_amdgcn_exp2f(m - top);
      l *= f;
#pragma unroll
      for (int d = 0; d < DT16; ++d) o[d] *= f;
      m = top;
    }
    const float ref = top == -INFINITY ? 0.f : top;
#pragma unroll
    for (int kt = 0; kt < 2; ++kt)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        s[kt][e] = __builtin_amdgcn_exp2f(s[kt][e] - ref);
        l += s[kt][e];
      }
    const Frag<T> pf = frag_of<T>(s[0], s[1]);
    __builtin_amdgcn_wave_barrier();
#pragma unroll
    for (int d = 0; d < DT16; ++d) {
      const Frag<T> a = frag_cols<T, TL::PITCH>(vs, 0, d * 16, lane);
      o[d] = attn_mma(o[d], a, pf);
      if constexpr (sizeof(T) == 2) o[d] = attn_mma(o[d], a, frag_rest<T>(s[0], s[1], pf));
    }
    __builtin_amdgcn_wave_barrier();
  }
  // join the waves (in wave order)
  l = cols_sum(l);
  if (g == 0) {
    ml[wave][c][0] = m;
    ml[wave][c][1] = l;
  }
  __syncthreads();
  float* os = reinterpret_cast<float*>(smem);
#pragma unroll
  for (int d = 0; d < DT16; ++d)
#pragma unroll
    for (int e = 0; e < 4; ++e) os[(wave * 16 + c) * (DP + 1) + d * 16 + g * 4 + e] = o[d][e];
  __syncthreads();
  for (int x = tid; x < 16 * DP; x += 256) {
    const int r = x / DP, d = x % DP, rr = rt * 16 + r;
    if (rr >= rows) continue;
    float top = -INFINITY, sum = 0.f, val = 0.f;
#pragma unroll
    for (int w = 0; w < 4; ++w) top = fmaxf(top, ml[w][r][0]);
    bool nan = false;
#pragma unroll
    for (int w = 0; w < 4; ++w) {
      const float f = ml[w][r][0] == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(ml[w][r][0] - top);
      nan |= ml[w][r][1] != ml[w][r][1];
      sum += ml[w][r][1] * f;
      val += os[(w * 16 + r) * (DP + 1) + d] * f;
    }
    if (nan) sum = val = NAN;
    const int qi = rr / share, hh = hk * share + rr - qi * share;
    const int64_t at = ((int64_t)b * p.H + hh) * p.Lq + qi;
    if (p.splits == 1) {
      if (d < p.D)
        store_o1(static_cast<T*>(p.o), static_cast<T*>(p.rest), (((int64_t)b * p.Lq + qi) * p.H + hh) * p.D + d, sum == 0.f ? 0.f : val / sum);
      if (d == 0 && p.lse) p.lse[at] = sum == 0.f ? -INFINITY : top + __builtin_amdgcn_logf(sum);
    } else {
      const int64_t n = (int64_t)p.B * p.H * p.Lq, slot = split * n + at;
      if (d < p.D) p.part[2 * p.splits * n + slot * p.D + d] = val;
      if (d == 0) {
        p.part[2 * slot] = top;
        p.part[2 * slot + 1] = sum;
      }
    }
  }
}

// A row's splits (64 at most), joined in a fixed order by a block: a lane holds a split's maximum and sum, then up to two columns of the result; the
// waves take every fourth split, so that a row waits for memory twice (32 splits of 32 x 16 rows, heads of 64: one wave to a row took 13.8 us, this 4.7).
template <typename T>
__global__ __launch_bounds__(256) void attn_join_kernel(const AttnParams p) {
  __shared__ float vals[4][128], weight[64];
  const int64_t n = (int64_t)p.B * p.H * p.Lq, at = blockIdx.x;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  float m = -INFINITY, l = 0.f;
  if (lane < p.splits) {
    m = p.part[2 * (lane * n + at)];
    l = p.part[2 * (lane * n + at) + 1];
  }
  const float top = wave_max(m), f = m == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(m - top), sum = wave_sum(l * f);
  if (wave == 0) weight[lane] = f;
  __syncthreads();
  const float* part = p.part + 2 * p.splits * n + at * p.D;
  const int c0 = min(lane, p.D - 1), c1 = min(lane + 64, p.D - 1);             // (in bounds; not stored below)
  float val[2] = {0.f, 0.f};
#pragma unroll 8
  for (int s = wave; s < p.splits; s += 4) {
    const float w = weight[s], a = part[s * n * p.D + c0], b = p.D > 64 ? part[s * n * p.D + c1] : 0.f;
    val[0] += w == 0.f ? 0.f : a * w;                                          // (a split without keys: its columns may hold NaN)
    val[1] += w == 0.f ? 0.f : b * w;
  }
  vals[wave][lane] = val[0];
  vals[wave][64 + lane] = val[1];
  __syncthreads();
  const int d = threadIdx.x, i = at % p.Lq, h = at / p.Lq % p.H, b = at / p.Lq / p.H;
  if (d < p.D)
    store_o1(static_cast<T*>(p.o), static_cast<T*>(p.rest), (((int64_t)b * p.Lq + i) * p.H + h) * p.D + d,
             sum == 0.f ? 0.f : sum == sum ? (((vals[0][d] + vals[1][d]) + vals[2][d]) + vals[3][d]) / sum : NAN);
  if (d == 0 && p.lse) p.lse[at] = sum == 0.f ? -INFINITY : top + __builtin_amdgcn_logf(sum);
}

// ----------------------------------------------------------------------------------------------------------------------------- backward
// dQ, delta and the sums of dS by bucket.  As the forward: a lane owns a query's column, K and V tiles stream through LDS; dQ^T += K^T dS^T.
// The sums by bucket go by distance first, since a distance is a diagonal of dS: 16 queries by 32 keys of dS are laid into the wave's corner of LDS with zeros around
// them, 47 lanes add a diagonal's 16 entries each and keep it in a table by distance (no two lanes share an entry, so results do not depend on any order); tiles
// wholly beyond `far` add into two registers instead.  (One LDS addition for each element by bucket took 66 us of 104 on 16 x 300 queries, 8 heads of 32; this takes 10.)
template <typename T, int DP, int NQ, int BK, bool MASK>
__global__ __launch_bounds__(256, 2) void attn_dq_kernel(const AttnParams p) {
  constexpr int KP = DP / 32, DT16 = DP / 16, BQ = 64 * NQ;
  using TL = Tile<T, DP, BK, 256>;
  extern __shared__ __attribute__((aligned(16))) unsigned char smem[];
  T* kt_ = reinterpret_cast<T*>(smem);
  T* vt_ = reinterpret_cast<T*>(smem + 2 * TL::BYTES);
  using ML = MaskTile<BQ, BK>;
  uint32_t* mt_ = reinterpret_cast<uint32_t*>(smem + 4 * TL::BYTES);
  float* bias = reinterpret_cast<float*>(smem + 4 * TL::BYTES + 2 * ML::BYTES);
  constexpr int DROW = 68, DIAG = 16 * DROW;                                   // the wave's corner: 16 zeros, 32 keys, 16 zeros and 4 to spread the banks
  const int entries = p.table ? (2 * p.far + 12) / 4 * 4 : 0, ends = 2 * p.far + 1;   // (whole 16 bytes)
  float* diag = bias + entries;                                                // [wave][16][DROW]
  float* by = diag + 4 * DIAG;                                                 // [wave][2 far + 1]: sums by distance
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), c = lane & 15, g = lane >> 4;
  const int id = xcd_order(blockIdx.x, gridDim.x);
  int bh, qt;
  tile_order(p, id, p.B * p.H, &bh, &qt);
  const int b = bh / p.H, h = bh - b * p.H, hk = h / (p.H / p.Hk);
  const Span sp = span_of(p, b, h);
  const T* kb = static_cast<const T*>(p.k) + b * p.k_sb + hk * p.k_sh;
  const T* vb = static_cast<const T*>(p.v) + b * p.v_sb + hk * p.v_sh;
  const int q0 = qt * BQ + wave * 16 * NQ;
  const int last = min(qt * BQ + BQ, p.Lq) - 1 + sp.start;
  const int kend = p.causal ? min(sp.klen, last + 1) : sp.klen;
  const int nt = kend > 0 ? (kend + BK - 1) / BK : 0;
  TL kr, vr;
  ML mr;
  if (nt > 0) {
    kr.load(kb, p.k_sl, 0, kend, p.D, MASK ? sp.hide : nullptr, tid);
    vr.load(vb, p.v_sl, 0, kend, p.D, MASK ? sp.hide : nullptr, tid);
    if constexpr (MASK) mr.load(sp.mask, sp.m_sq, qt * BQ, p.Lq, 0, p.Lk, tid);
  }
  Frag<T> qf[NQ][KP], gf[NQ][KP];
  float lse[NQ], delta[NQ];
#pragma unroll
  for (int n = 0; n < NQ; ++n) {
    const int i = q0 + n * 16 + c;
    const bool in = i < p.Lq;
    const T* qp = static_cast<const T*>(p.q) + b * p.q_sb + (int64_t)i * p.q_sl + h * p.q_sh + g * 8;
    const T* gp = static_cast<const T*>(p.dout) + b * p.g_sb + (int64_t)i * p.g_sl + h * p.g_sh + g * 8;
    const int64_t oat = (((int64_t)b * p.Lq + i) * p.H + h) * p.D + g * 8;
    const T *op = static_cast<const T*>(p.o) + oat, *rp = static_cast<const T*>(p.rest) + oat;
    // delta = the diagonal of O dO^T by the same products as dP = V dO^T: where one key holds all the weight, O is its value and dS exactly zero
    f32x4 od = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int kp = 0; kp < KP; ++kp) {
      const bool on = in && kp * 32 + g * 8 < p.D;
      qf[n][kp] = on ? frag_row(qp + kp * 32) : frag_zero<T>();
      gf[n][kp] = on ? frag_row(gp + kp * 32) : frag_zero<T>();
      od = attn_mma(od, on ? frag_row(op + kp * 32) : frag_zero<T>(), gf[n][kp]);
    }
    if (p.rest) {
#pragma unroll
      for (int kp = 0; kp < KP; ++kp) od = attn_mma(od, in && kp * 32 + g * 8 < p.D ? frag_row(rp + kp * 32) : frag_zero<T>(), gf[n][kp]);
    }
    const float mine = (c & 2) ? ((c & 1) ? od.w : od.z) : ((c & 1) ? od.y : od.x);
    delta[n] = __shfl(mine, (c >> 2) * 16 + c);
    const int64_t at = ((int64_t)b * p.H + h) * p.Lq + i;
    lse[n] = in ? p.lse[at] : INFINITY;
    if (lse[n] == -INFINITY) lse[n] = INFINITY;                                // an empty row: every probability 0
    if (in && g == 0) p.delta[at] = delta[n];
  }
  f32x4 dq[DT16][NQ];
#pragma unroll
  for (int n = 0; n < NQ; ++n)
#pragma unroll
    for (int d = 0; d < DT16; ++d) dq[d][n] = f32x4{0.f, 0.f, 0.f, 0.f};
  float* corner = diag + wave * DIAG;
  float* mine = by + wave * ends;
  float before = 0.f, after = 0.f;
  if (p.table) load_bias<T>(p, h, bias, 256);
  if (p.part) {
    for (int e = lane; e < DIAG; e += 64) corner[e] = 0.f;
    for (int e = lane; e < ends; e += 64) mine[e] = 0.f;
  }
  if (nt > 0) {
    kr.store(kt_, tid);
    vr.store(vt_, tid);
    if constexpr (MASK) mr.store(mt_, 0, p.Lk, tid);
  }
  __syncthreads();
  for (int t = 0; t < nt; ++t) {
    const T* ks = kt_ + (t & 1) * (TL::BYTES / (int)sizeof(T));
    const T* vs = vt_ + (t & 1) * (TL::BYTES / (int)sizeof(T));
    const uint32_t* ms = mt_ + (t & 1) * (ML::BYTES / 4);
    const int j0 = t * BK;
    if (t + 1 < nt) {
      kr.load(kb, p.k_sl, j0 + BK, kend, p.D, MASK ? sp.hide : nullptr, tid);
      vr.load(vb, p.v_sl, j0 + BK, kend, p.D, MASK ? sp.hide : nullptr, tid);
      if constexpr (MASK) mr.load(sp.mask, sp.m_sq, qt * BQ, p.Lq, j0 + BK, p.Lk, tid);
    }
    const int p0 = q0 + sp.start, p1 = p0 + 16 * NQ - 1;
    const int far = p.table ? beyond(j0, BK, p0, p1, p.far) : -1;
    const bool cut = MASK || j0 + BK > sp.klen || (p.causal && j0 + BK - 1 > p0);
    const float fixed = p.table && far ? bias[far < 0 ? 0 : 2 * p.far + 8] : 0.f;
    float sum = 0.f;
#pragma unroll
    for (int kc = 0; kc < BK / 32; ++kc) {                                     // 32 keys at a time: two score tiles make one operand
      f32x4 s[2][NQ], w[2][NQ];
#pragma unroll
      for (int kt = 0; kt < 2; ++kt) {
#pragma unroll
        for (int n = 0; n < NQ; ++n) s[kt][n] = w[kt][n] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int kp = 0; kp < KP; ++kp) {
          const int off = (kc * 32 + kt * 16 + c) * TL::PITCH + kp * 32 + g * 8;
          const Frag<T> a = frag_row(ks + off), v = frag_row(vs + off);
#pragma unroll
          for (int n = 0; n < NQ; ++n) {
            s[kt][n] = attn_mma(s[kt][n], a, qf[n][kp]);
            w[kt][n] = attn_mma(w[kt][n], v, gf[n][kp]);
          }
        }
      }
      Frag<T> df[NQ];
#pragma unroll
      for (int n = 0; n < NQ; ++n) {
        const int i = q0 + n * 16 + c, pos = i + sp.start;
        const int end = p.causal ? min(sp.klen, pos + 1) : sp.klen;
        uint32_t off = 0u;
        if (cut) {
          off = past_bits(end - j0 - kc * 32);
          if constexpr (MASK) off |= ms[(wave * 16 * NQ + n * 16 + c) * ML::WORDS + kc];
          off >>= 4 * g;
        }
#pragma unroll
        for (int kt = 0; kt < 2; ++kt) {
          const int j = j0 + kc * 32 + kt * 16 + 4 * g;
          f32x4 add = f32x4{fixed, fixed, fixed, fixed} - lse[n];
          if (!far) add = bias4(bias + bias_at(j - pos, p.far)) - lse[n];
#pragma unroll
          for (int e = 0; e < 4; ++e)                                          // scale, bias and the row's statistic in one multiply-add
            s[kt][n][e] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[kt][n][e], p.scale2, add[e])) * (w[kt][n][e] - delta[n]);
          if (cut) {
#pragma unroll
            for (int e = 0; e < 4; ++e) s[kt][n][e] = pick(bit_mask(off, kt * 16 + e), 0.f, s[kt][n][e]);
          }
          if (far) sum += (s[kt][n].x + s[kt][n].y) + (s[kt][n].z + s[kt][n].w);
          else if (p.part) *reinterpret_cast<f32x4*>(corner + c * DROW + 16 + kt * 16 + 4 * g) = s[kt][n];
        }
        if (p.part && !far) {
          __builtin_amdgcn_wave_barrier();
          float v = 0.f;
#pragma unroll
          for (int x = 0; x < 16; ++x) v += lane < 48 ? corner[x * (DROW + 1) + lane] : 0.f;   // diagonal key - query = lane - 16
          const int dist = j0 + kc * 32 - (q0 + n * 16 + sp.start) + lane - 16;
          if (dist <= -p.far) before += v;
          else if (dist >= p.far) after += v;
          else if (lane < 48) mine[dist + p.far] += v;
          __builtin_amdgcn_wave_barrier();
        }
        df[n] = frag_of<T>(s[0][n], s[1][n]);
      }
#pragma unroll
      for (int d = 0; d < DT16; ++d) {
        const Frag<T> a = frag_cols<T, TL::PITCH>(ks, kc * 32, d * 16, lane);
#pragma unroll
        for (int n = 0; n < NQ; ++n) dq[d][n] = attn_mma(dq[d][n], a, df[n]);
      }
    }
    before += far < 0 ? sum : 0.f;
    after += far > 0 ? sum : 0.f;
    if (t + 1 < nt) {
      kr.store(kt_ + ((t + 1) & 1) * (TL::BYTES / (int)sizeof(T)), tid);
      vr.store(vt_ + ((t + 1) & 1) * (TL::BYTES / (int)sizeof(T)), tid);
      if constexpr (MASK) mr.store(mt_ + ((t + 1) & 1) * (ML::BYTES / 4), j0 + BK, p.Lk, tid);
    }
    __syncthreads();
  }
  if (p.dq) {
#pragma unroll
    for (int n = 0; n < NQ; ++n) {
      const int i = q0 + n * 16 + c;
      if (i >= p.Lq) continue;
      T* op = static_cast<T*>(p.dq) + (((int64_t)b * p.Lq + i) * p.H + h) * p.D + g * 4;
#pragma unroll
      for (int d = 0; d < DT16; ++d)
        if (d * 16 + g * 4 < p.D) DT<T>::store4(op + d * 16, dq[d][n] * p.scale);
    }
  }
  if (p.part) {
    before = wave_sum(before);
    after = wave_sum(after);
    if (lane == 0) {
      mine[0] = before;
      mine[ends - 1] = after;
    }
    __syncthreads();
    int* place = reinterpret_cast<int*>(diag);                                 // (the corners are free now)
    for (int e = tid; e < ends; e += 256) {
      by[e] = ((by[e] + by[ends + e]) + by[2 * ends + e]) + by[3 * ends + e];
      place[e] = min((int)p.lut[e], p.nb - 1);
    }
    __syncthreads();
    float* out = p.part + ((int64_t)h * p.B * p.tiles + (int64_t)b * p.tiles + qt) * p.nb;
    for (int k = wave; k < p.nb; k += 4) {                                     // a wave adds the distances of a bucket
      float v = 0.f;
#pragma unroll 4
      for (int e = lane; e < ends; e += 64) v += place[e] == k ? by[e] : 0.f;
      v = wave_sum(v);
      if (lane == 0) out[k] = v;
    }
  }
}

// dtable[k][h] = the blocks' sums added in block order: a wave to a (bucket, head)
template <typename T>
__global__ __launch_bounds__(256) void attn_dtable_kernel(const float* __restrict__ part, int nb, int H, int blocks, T* __restrict__ dtable) {
  const int x = blockIdx.x * 4 + (threadIdx.x >> 6), lane = threadIdx.x & 63;
  if (x >= nb * H) return;
  const int h = x / nb, k = x - h * nb;
  float v = 0.f;
  for (int s = lane; s < blocks; s += 64) v += part[((int64_t)h * blocks + s) * nb + k];
  v = wave_sum(v);
  if (lane == 0) DT<T>::store1(dtable + (int64_t)k * H + h, v);
}

// dK and dV.  A lane owns a key's column (K and V of it in registers as operands), Q and dO tiles stream through LDS with their rows' lse and delta:
// S = Q K^T, dP = dO V^T, then dV^T += dO^T P and dK^T += Q^T dS.  The heads that share the keys follow one another, so their sum needs no atomics.
template <typename T, int DP, int NK, int BQ, bool MASK>
__global__ __launch_bounds__(256, 2) void attn_dkv_kernel(const AttnParams p) {
  constexpr int KP = DP / 32, DT16 = DP / 16, BKB = 64 * NK;
  using TL = Tile<T, DP, BQ, 256>;
  extern __shared__ __attribute__((aligned(16))) unsigned char smem[];
  T* qt_ = reinterpret_cast<T*>(smem);
  T* gt_ = reinterpret_cast<T*>(smem + 2 * TL::BYTES);
  using ML = MaskTile<BQ, BKB>;
  uint32_t* mt_ = reinterpret_cast<uint32_t*>(smem + 4 * TL::BYTES);
  float* stat = reinterpret_cast<float*>(smem + 4 * TL::BYTES + 2 * ML::BYTES);   // [2][lse BQ | delta BQ]
  float* bias = stat + 4 * BQ;
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), c = lane & 15, g = lane >> 4;
  const int id = xcd_order(blockIdx.x, gridDim.x);
  int bh, jt;
  tile_order(p, id, p.B * p.Hk, &bh, &jt);
  jt = p.tiles - 1 - jt;                                                       // (the first keys are seen by the most queries)
  const int b = bh / p.Hk, hk = bh - b * p.Hk, share = p.H / p.Hk;
  const int jb = jt * BKB, jw = jb + wave * 16 * NK;                           // the block's and the wave's first key
  const Span sp = span_of(p, b, hk * share);
  const int kall = p.causal ? min(sp.klen, p.Lq + sp.start) : sp.klen;         // (no query sees a key from here on)
  const T* kb = static_cast<const T*>(p.k) + b * p.k_sb + hk * p.k_sh;
  const T* vb = static_cast<const T*>(p.v) + b * p.v_sb + hk * p.v_sh;
  Frag<T> kf[NK][KP], vf[NK][KP];
#pragma unroll
  for (int n = 0; n < NK; ++n) {
    const int j = jw + n * 16 + c;
    const bool in = j < kall && !(MASK && sp.hide && p.m_sh == 0 && sp.hide[j]);
#pragma unroll
    for (int kp = 0; kp < KP; ++kp) {
      const bool on = in && kp * 32 + g * 8 < p.D;
      kf[n][kp] = on ? frag_row(kb + (int64_t)j * p.k_sl + kp * 32 + g * 8) : frag_zero<T>();
      vf[n][kp] = on ? frag_row(vb + (int64_t)j * p.v_sl + kp * 32 + g * 8) : frag_zero<T>();
    }
  }
  f32x4 dk[DT16][NK], dv[DT16][NK];
#pragma unroll
  for (int n = 0; n < NK; ++n)
#pragma unroll
    for (int d = 0; d < DT16; ++d) dk[d][n] = dv[d][n] = f32x4{0.f, 0.f, 0.f, 0.f};
  // queries that see a key of this block: from the one at its first key's position on
  const int i0 = p.causal ? max(0, jb - sp.start) / BQ * BQ : 0;
  const int nt = jb < sp.klen && i0 < p.Lq ? (p.Lq - i0 + BQ - 1) / BQ : 0, all = nt * share;
  TL qr, gr;
  ML mr;
  float st = 0.f;
  auto load = [&](int t) {                                                     // tile t: head t / nt of the group, queries i0 + (t % nt) BQ ..
    const int h = hk * share + t / nt, i = i0 + (t % nt) * BQ;
    qr.load(static_cast<const T*>(p.q) + b * p.q_sb + h * p.q_sh, p.q_sl, i, p.Lq, p.D, nullptr, tid);
    gr.load(static_cast<const T*>(p.dout) + b * p.g_sb + h * p.g_sh, p.g_sl, i, p.Lq, p.D, nullptr, tid);
    if constexpr (MASK) mr.load(sp.mask + t / nt * p.m_sh, sp.m_sq, i, p.Lq, jb, p.Lk, tid);
    if (tid < 2 * BQ) {
      const int ii = i + tid % BQ;
      const float* src = tid < BQ ? p.lse : p.delta;
      st = ii < p.Lq ? src[((int64_t)b * p.H + h) * p.Lq + ii] : 0.f;
      if (tid < BQ) st = ii >= p.Lq || st == -INFINITY ? INFINITY : st - P_UP_LOG2<T>;   // no such row, or an empty one: every probability 0
      else st *= 1.f / P_UP<T>;
    }
  };
  auto keep = [&](int t) {
    qr.store(qt_ + (t & 1) * (TL::BYTES / (int)sizeof(T)), tid);
    gr.store(gt_ + (t & 1) * (TL::BYTES / (int)sizeof(T)), tid);
    if constexpr (MASK) mr.store(mt_ + (t & 1) * (ML::BYTES / 4), jb, p.Lk, tid);
    if (tid < 2 * BQ) stat[(t & 1) * 2 * BQ + tid] = st;
  };
  if (all > 0) {
    load(0);
    if (p.table) load_bias<T>(p, hk * share, bias, 256);
    keep(0);
  }
  __syncthreads();
  for (int t = 0; t < all; ++t) {
    const int h = hk * share + t / nt, iq = i0 + (t % nt) * BQ;
    if (t && t % nt == 0) {                                                    // the next head of the group: its bias, its mask
      if (p.table) {
        load_bias<T>(p, h, bias, 256);
        __syncthreads();
      }
    }
    const uint32_t* ms = mt_ + (t & 1) * (ML::BYTES / 4) + wave * NK / 2;      // (the words of the wave's keys)
    const T* qs = qt_ + (t & 1) * (TL::BYTES / (int)sizeof(T));
    const T* gs = gt_ + (t & 1) * (TL::BYTES / (int)sizeof(T));
    const float* ls = stat + (t & 1) * 2 * BQ;
    if (t + 1 < all) load(t + 1);
    const int p0 = iq + sp.start, p1 = p0 + BQ - 1;
    const int far = p.table ? beyond(jw, 16 * NK, p0, p1, p.far) : -1;
    const bool cut = MASK || jw + 16 * NK > sp.klen || (p.causal && jw + 16 * NK - 1 > p0);
    const float fixed = p.table && far ? bias[far < 0 ? 0 : 2 * p.far + 8] : 0.f;
#pragma unroll
    for (int qc = 0; qc < BQ / 32; ++qc) {
      f32x4 s[2][NK], w[2][NK];
#pragma unroll
      for (int qq = 0; qq < 2; ++qq) {
#pragma unroll
        for (int n = 0; n < NK; ++n) s[qq][n] = w[qq][n] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int kp = 0; kp < KP; ++kp) {
          const int off = (qc * 32 + qq * 16 + c) * TL::PITCH + kp * 32 + g * 8;
          const Frag<T> a = frag_row(qs + off), x = frag_row(gs + off);
#pragma unroll
          for (int n = 0; n < NK; ++n) {
            s[qq][n] = attn_mma(s[qq][n], a, kf[n][kp]);
            w[qq][n] = attn_mma(w[qq][n], x, vf[n][kp]);
          }
        }
      }
      Frag<T> pf[NK], df[NK];
#pragma unroll
      for (int qq = 0; qq < 2; ++qq) {
        const int i = qc * 32 + qq * 16 + 4 * g;                               // the lane's first of four queries in the tile
        const f32x4 ll = *reinterpret_cast<const f32x4*>(ls + i), dd = *reinterpret_cast<const f32x4*>(ls + BQ + i);
        uint32_t hid[4] = {0u, 0u, 0u, 0u};
        if constexpr (MASK) {
#pragma unroll
          for (int e = 0; e < 4; ++e) hid[e] = ms[(i + e) * ML::WORDS] >> ((wave * NK & 1) * 16 + c);
        }
#pragma unroll
        for (int n = 0; n < NK; ++n) {
          const int j = jw + n * 16 + c, pos = p0 + i;
          f32x4 add = f32x4{fixed, fixed, fixed, fixed} - ll;
          if (!far) {
            const f32x4 w4 = bias4(bias + bias_at(j - pos - 3, p.far));          // four neighbours, the last query's first
            add = f32x4{w4.w, w4.z, w4.y, w4.x} - ll;
          }
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            s[qq][n][e] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[qq][n][e], p.scale2, add[e]));
            w[qq][n][e] = s[qq][n][e] * __builtin_fmaf(w[qq][n][e], 1.f / P_UP<T>, -dd[e]);
          }
          if (cut) {
            const uint32_t off = j >= sp.klen ? 15u : p.causal ? ~past_bits(j - pos) : 0u;   // (bit e: the key lies behind query e)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const uint32_t none = bit_mask(off, e) | bit_mask(hid[e], n * 16);
              s[qq][n][e] = pick(none, 0.f, s[qq][n][e]);
              w[qq][n][e] = pick(none, 0.f, w[qq][n][e]);
            }
          }
        }
      }
#pragma unroll
      for (int n = 0; n < NK; ++n) {
        pf[n] = frag_of<T>(s[0][n], s[1][n]);
        df[n] = frag_of<T>(w[0][n], w[1][n]);
      }
#pragma unroll
      for (int d = 0; d < DT16; ++d) {
        const Frag<T> a = frag_cols<T, TL::PITCH>(gs, qc * 32, d * 16, lane), x = frag_cols<T, TL::PITCH>(qs, qc * 32, d * 16, lane);
#pragma unroll
        for (int n = 0; n < NK; ++n) {
          dv[d][n] = attn_mma(dv[d][n], a, pf[n]);
          dk[d][n] = attn_mma(dk[d][n], x, df[n]);
        }
      }
    }
    if (t + 1 < all) keep(t + 1);
    __syncthreads();
  }
#pragma unroll
  for (int n = 0; n < NK; ++n) {
    const int j = jw + n * 16 + c;
    if (j >= p.Lk) continue;
    const int64_t at = (((int64_t)b * p.Lk + j) * p.Hk + hk) * p.D + g * 4;
#pragma unroll
    for (int d = 0; d < DT16; ++d)
      if (d * 16 + g * 4 < p.D) {
        if (p.dk) DT<T>::store4(static_cast<T*>(p.dk) + at + d * 16, dk[d][n] * p.scale);
        if (p.dv) DT<T>::store4(static_cast<T*>(p.dv) + at + d * 16, dv[d][n] * (1.f / P_UP<T>));
      }
  }
}

// -------------------------------------------------------------------------------------------------------------------------------- host
static bool attn_stride_ok(int64_t s, int es) { return s >= 0 && s * es % 16 == 0; }

// The keys are split where there are few rows, or too few blocks of 64 queries to fill the chip, and keys enough to pay for the join (us, split against whole: bf16
// heads of 64, 8 x 8 heads over 2, 4 queries, 4096 keys 13.0 / 72; 8 heads, 64 queries, 4096 keys 16.5 / 72, 1024 keys 11.8 / 20.6, 300 keys 11.5 / 9.2; 64 x 8 heads, 16 queries,
// 1024 keys 46.5 / 43.4; 512 x 8 heads of 32, 8 queries, 300 keys 64 / 43; fp32, whose products take longer, 3 x 6 heads of 40, 77 queries, 401 keys 14.8 / 26).
static bool attn_uses_split(const moy_attention_args* a) {
  if (a->Lk < (a->dtype == MOY_F32 ? 256 : 512)) return false;
  return (int64_t)a->Lq * (a->H / a->Hk) <= 16 || (int64_t)a->B * a->H * ((a->Lq + 63) / 64) < 128;
}

// Splits of at least 256 keys (two 32-key tiles to a wave), as many as give sixteen blocks to a compute unit, of which four fit at a time: sequences differ in
// length, and what follows fills in (32 caches of up to 16384 keys, 4 key heads of 64: 90.6 us with four blocks, 84.7 with eight, 77.6 with sixteen).  64 at most.
static void attn_splits(const moy_attention_args* a, int* tiles, int* splits, int* keys) {
  const int rows = a->Lq * (a->H / a->Hk);
  *tiles = (rows + 15) / 16;
  const int64_t blocks = (int64_t)a->B * a->Hk * *tiles;
  int64_t s = (4096 + blocks - 1) / blocks;
  const int64_t most = (a->Lk + 255) / 256;
  if (s > most) s = most;
  if (s > 64) s = 64;
  *keys = (int)(((a->Lk + s - 1) / s + 127) / 128 * 128);
  *splits = (a->Lk + *keys - 1) / *keys;
}

static int attn_check(const moy_attention_args* a, bool bwd) {
  if (!a || a->dtype < MOY_F32 || a->dtype > MOY_F16) return MOY_EINVAL;
  const int es = a->dtype == MOY_F32 ? 4 : 2;
  if (!a->q || !a->k || !a->v || !a->o || a->B <= 0 || a->H <= 0 || a->Hk <= 0 || a->Lq <= 0 || a->Lk <= 0 || a->D <= 0) return MOY_EINVAL;
  if (a->H % a->Hk || a->D % 8) return MOY_EINVAL;
  if (a->D > 128) return MOY_ENOSYS;
  if (a->Lq > (1 << 29) || a->Lk > (1 << 29) || a->q_start > (1 << 30) || a->q_start < -(1 << 30)) return MOY_EINVAL;
  if (!aligned16(a->q) || !aligned16(a->k) || !aligned16(a->v) || !aligned16(a->o)) return MOY_EINVAL;
  const int64_t st[] = {a->q_sb, a->q_sl, a->q_sh, a->k_sb, a->k_sl, a->k_sh, a->v_sb, a->v_sl, a->v_sh};
  for (int64_t s : st)
    if (!attn_stride_ok(s, es)) return MOY_EINVAL;
  if ((a->table == nullptr) != (a->lut == nullptr)) return MOY_EINVAL;
  if (a->table && (a->num_buckets < 1 || a->num_buckets > 64 || a->max_distance < 1 || a->max_distance > 1024)) return MOY_EINVAL;
  if (reinterpret_cast<uintptr_t>(a->table) % es || reinterpret_cast<uintptr_t>(a->k_len) % 4) return MOY_EINVAL;
  if (a->mask && (a->m_sb < 0 || a->m_sh < 0 || a->m_sq < 0)) return MOY_EINVAL;
  if (!(a->scale >= 0.f) || !(a->scale - a->scale == 0.f) || (a->o_rest && !aligned16(a->o_rest))) return MOY_EINVAL;
  if ((int64_t)a->B * a->H > (1 << 24) || (int64_t)a->B * a->H * ((a->Lq > a->Lk ? a->Lq : a->Lk) / 64 + 1) > 0x7fffffffLL / 8) return MOY_EINVAL;
  // every launch has a grid that can be launched
  const int64_t heads = (int64_t)a->B * a->H, groups = (int64_t)a->B * a->Hk;
  if (!bwd && attn_uses_split(a)) {
    int tiles, splits, keys;
    attn_splits(a, &tiles, &splits, &keys);
    if (!grid_fits(groups * tiles * splits, 256) || !grid_fits(heads * a->Lq, 256)) return MOY_ENOSYS;
  } else if (!grid_fits(heads * ((a->Lq + 63) / 64), 256) || (bwd && !grid_fits(groups * ((a->Lk + 63) / 64), 256))) {
    return MOY_ENOSYS;
  }
  if (bwd) {
    const int64_t gs[] = {a->g_sb, a->g_sl, a->g_sh};
    for (int64_t s : gs)
      if (!attn_stride_ok(s, es)) return MOY_EINVAL;
    if (!a->lse || !a->dout || !aligned16(a->dout) || !aligned16(a->dq) || !aligned16(a->dk) || !aligned16(a->dv)) return MOY_EINVAL;
    if (!a->dq && !a->dk && !a->dv && !a->dtable) return MOY_EINVAL;
    if (a->dtable && (!a->table || reinterpret_cast<uintptr_t>(a->dtable) % es)) return MOY_EINVAL;
  }
  return MOY_OK;
}

static AttnParams attn_params(const moy_attention_args* a) {
  AttnParams p{};
  p.q = a->q; p.k = a->k; p.v = a->v;
  p.q_sb = a->q_sb; p.q_sl = a->q_sl; p.q_sh = a->q_sh; p.k_sb = a->k_sb; p.k_sl = a->k_sl; p.k_sh = a->k_sh;
  p.v_sb = a->v_sb; p.v_sl = a->v_sl; p.v_sh = a->v_sh;
  p.B = a->B; p.H = a->H; p.Hk = a->Hk; p.Lq = a->Lq; p.Lk = a->Lk; p.D = a->D;
  p.table = a->table; p.lut = a->lut; p.nb = a->num_buckets; p.far = a->max_distance;
  p.k_len = a->k_len; p.q_from_end = a->q_from_end; p.q_start = a->q_start; p.causal = a->causal;
  p.mask = a->mask; p.m_sb = a->m_sb; p.m_sh = a->m_sh; p.m_sq = a->m_sq;
  p.scale = a->scale; p.scale2 = a->scale * LOG2E;
  p.o = a->o; p.lse = a->lse;
  p.rest = a->dtype == MOY_F32 ? nullptr : a->o_rest;
  p.dout = a->dout; p.g_sb = a->g_sb; p.g_sl = a->g_sl; p.g_sh = a->g_sh;
  p.dq = a->dq; p.dk = a->dk; p.dv = a->dv;
  return p;
}

static size_t attn_bias_bytes(const moy_attention_args* a) { return a->table ? (2 * (size_t)a->max_distance + 12) / 4 * 16 : 0; }

// 16-bit heads of 40 to 64: 32 queries (keys) to a wave where that leaves two blocks to a compute unit (8 x 1024 x 8 heads of 64: forward 43 us against 48, dQ
// 88 against 102, dK and dV 61 against 75; 2 x 1024 x 16, half the blocks: 33.5 against 28, 68 against 54, 54 against 41), 16 otherwise; heads up to 32 have
// the registers for twice the waves and are faster with 16 at any size (64 x 300 x 8: 33.9 against 31.4, 50.7 against 45.1).
static bool attn_wide(const moy_attention_args* a, int heads, int rows) { return (int64_t)a->B * heads * ((rows + 127) / 128) >= 512; }

template <typename T, int DP, int NQ, bool MASK>
static int attn_fwd_tiles(const moy_attention_args* a, AttnParams p, hipStream_t st) {
  constexpr int BK = attn_bk<T, DP>();
  auto kern = attn_fwd_kernel<T, DP, NQ, BK, MASK>;
  static std::atomic<uint64_t> ready{0};
  const int rc = lds_opt_in(reinterpret_cast<const void*>(kern), ready);
  if (rc != MOY_OK) return rc;
  p.tiles = (a->Lq + 64 * NQ - 1) / (64 * NQ);
  const size_t lds = 4 * Tile<T, DP, BK, 256>::BYTES + 2 * MaskTile<64 * NQ, BK>::BYTES + attn_bias_bytes(a);
  hipLaunchKernelGGL(kern, dim3((unsigned)(a->B * a->H * p.tiles)), dim3(256), lds, st, p);
  return launch_status();
}

template <typename T, int DP, bool MASK>
static int attn_fwd(const moy_attention_args* a, AttnParams p, hipStream_t st) {
  if (attn_uses_split(a)) {
    attn_splits(a, &p.tiles, &p.splits, &p.split_keys);
    p.part = a->ws;
    hipLaunchKernelGGL((attn_split_kernel<T, DP>), dim3((unsigned)((int64_t)a->B * a->Hk * p.tiles * p.splits)), dim3(256), 0, st, p);
    const int rc = launch_status();
    if (rc != MOY_OK || p.splits == 1) return rc;
    hipLaunchKernelGGL((attn_join_kernel<T>), dim3((unsigned)((int64_t)a->B * a->H * a->Lq)), dim3(256), 0, st, p);
    return launch_status();
  }
  if constexpr (sizeof(T) == 2 && DP == 64) {
    if (attn_wide(a, a->H, a->Lq)) return attn_fwd_tiles<T, DP, 2, MASK>(a, p, st);
  }
  return attn_fwd_tiles<T, DP, 1, MASK>(a, p, st);
}

template <typename T, int DP, int NQ, bool MASK>
static int attn_dq(const moy_attention_args* a, AttnParams p, hipStream_t st) {
  constexpr int BK = attn_bk<T, DP>();
  auto kern = attn_dq_kernel<T, DP, NQ, BK, MASK>;
  static std::atomic<uint64_t> ready{0};
  const int rc = lds_opt_in(reinterpret_cast<const void*>(kern), ready);
  if (rc != MOY_OK) return rc;
  const size_t bias = attn_bias_bytes(a), lds = 4 * Tile<T, DP, BK, 256>::BYTES + 2 * MaskTile<64 * NQ, BK>::BYTES + bias + (p.part ? 4 * 4 * (16 * 68 + 2 * (size_t)a->max_distance + 1) : 0);
  p.tiles = (a->Lq + 64 * NQ - 1) / (64 * NQ);
  hipLaunchKernelGGL(kern, dim3((unsigned)(a->B * a->H * p.tiles)), dim3(256), lds, st, p);
  return launch_status();
}

template <typename T, int DP, int NK, bool MASK>
static int attn_dkv(const moy_attention_args* a, AttnParams p, hipStream_t st) {
  constexpr int BQ = attn_bk<T, DP>();
  auto kern = attn_dkv_kernel<T, DP, NK, BQ, MASK>;
  static std::atomic<uint64_t> ready{0};
  const int rc = lds_opt_in(reinterpret_cast<const void*>(kern), ready);
  if (rc != MOY_OK) return rc;
  const size_t lds = 4 * Tile<T, DP, BQ, 256>::BYTES + 2 * MaskTile<BQ, 64 * NK>::BYTES + 16 * BQ + attn_bias_bytes(a);
  p.tiles = (a->Lk + 64 * NK - 1) / (64 * NK);
  hipLaunchKernelGGL(kern, dim3((unsigned)(a->B * a->Hk * p.tiles)), dim3(256), lds, st, p);
  return launch_status();
}

static int attn_dq_tiles(const moy_attention_args* a) {
  const int rows = a->dtype != MOY_F32 && a->D > 32 && a->D <= 64 && attn_wide(a, a->H, a->Lq) ? 128 : 64;
  return (a->Lq + rows - 1) / rows;
}

template <typename T, int DP, bool MASK>
static int attn_bwd(const moy_attention_args* a, AttnParams p, hipStream_t st) {
  int rc = MOY_ENOSYS;
  if constexpr (sizeof(T) == 2 && DP == 64) {
    if (attn_wide(a, a->H, a->Lq)) rc = attn_dq<T, DP, 2, MASK>(a, p, st);
  }
  if (rc == MOY_ENOSYS) rc = attn_dq<T, DP, 1, MASK>(a, p, st);
  if (rc != MOY_OK) return rc;
  if (a->dtable) {
    hipLaunchKernelGGL((attn_dtable_kernel<T>), dim3((a->num_buckets * a->H + 3) / 4), dim3(256), 0, st, p.part, a->num_buckets, a->H,
                       a->B * attn_dq_tiles(a), static_cast<T*>(a->dtable));
    if ((rc = launch_status()) != MOY_OK) return rc;
  }
  if (!a->dk && !a->dv) return MOY_OK;
  if constexpr (sizeof(T) == 2 && DP == 64) {
    if (attn_wide(a, a->Hk, a->Lk)) return attn_dkv<T, DP, 2, MASK>(a, p, st);
  }
  return attn_dkv<T, DP, 1, MASK>(a, p, st);
}

#define MOY_ATTN_HEADS(FN, T, ...)                                                                                              \
  (a->mask ? (a->D <= 32 ? FN<T, 32, true>(__VA_ARGS__) : a->D <= 64 ? FN<T, 64, true>(__VA_ARGS__) : FN<T, 128, true>(__VA_ARGS__))             \
           : (a->D <= 32 ? FN<T, 32, false>(__VA_ARGS__) : a->D <= 64 ? FN<T, 64, false>(__VA_ARGS__) : FN<T, 128, false>(__VA_ARGS__)))
#define MOY_ATTN_DISPATCH(FN, ...)                                                                                            \
  switch (a->dtype) {                                                                                                         \
    case MOY_F32: return MOY_ATTN_HEADS(FN, float, __VA_ARGS__);                                                              \
    case MOY_BF16: return MOY_ATTN_HEADS(FN, bf16_t, __VA_ARGS__);                                                            \
    default: return MOY_ATTN_HEADS(FN, f16_t, __VA_ARGS__);                                                                   \
  }

}  // namespace moy

using namespace moy;

extern "C" int64_t moy_attention_ws(const moy_attention_args* a) {
  const int rc = attn_check(a, false);
  if (rc != MOY_OK) return rc;
  if (!attn_uses_split(a)) return 0;
  int tiles, splits, keys;
  attn_splits(a, &tiles, &splits, &keys);
  return splits == 1 ? 0 : (int64_t)splits * a->B * a->H * a->Lq * (2 + a->D);
}

extern "C" int moy_attention(const moy_attention_args* a, void* stream) {
  const int64_t need = moy_attention_ws(a);
  if (need < 0) return (int)need;
  if (need > 0 && (!a->ws || a->ws_len < need)) return MOY_EINVAL;
  const AttnParams p = attn_params(a);
  hipStream_t st = static_cast<hipStream_t>(stream);
  MOY_ATTN_DISPATCH(attn_fwd, a, p, st)
}

extern "C" int64_t moy_attention_bwd_ws(const moy_attention_args* a) {
  const int rc = attn_check(a, true);
  if (rc != MOY_OK) return rc;
  return (int64_t)a->B * a->H * a->Lq + (a->dtable ? (int64_t)a->H * a->B * attn_dq_tiles(a) * a->num_buckets : 0);
}

extern "C" int moy_attention_bwd(const moy_attention_args* a, void* stream) {
  const int64_t need = moy_attention_bwd_ws(a);
  if (need < 0) return (int)need;
  if (!a->ws || a->ws_len < need) return MOY_EINVAL;
  AttnParams p = attn_params(a);
  p.delta = a->ws;
  p.part = a->dtable ? a->ws + (int64_t)a->B * a->H * a->Lq : nullptr;
  hipStream_t st = static_cast<hipStream_t>(stream);
  MOY_ATTN_DISPATCH(attn_bwd, a, p, st)
}
