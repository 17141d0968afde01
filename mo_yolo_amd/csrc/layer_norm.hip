// Layer norm as an operator of its own, forward and backward (nn.LayerNorm of the decoder layers and of QIM: nn/modules/transformer.py:515-652,
// MOTR/models/qim.py:73-340).  The inference kernels carry the norm in their epilogues; these are the forms that a training step needs.
//
//   s = x (+ r)   mu = mean(s)   v = mean((s - mu)^2)   xh = (s - mu) / sqrt(v + eps)   y = xh w + b
//   g = dy w      dx = dr = rstd (g - mean(g) - xh mean(g xh))       dw = sum_rows dy xh       db = sum_rows dy
//
// Both are bound by memory: forward reads x (and r) and writes y, backward reads dy and x (and r) and writes dx, each once.  A row lives in the
// registers of TPR lanes (NV chunks of 16 bytes each), so mean, centred variance and result are three sweeps over registers, and the variance
// never cancels.  Blocks walk the rows (a grid of about four blocks to a compute unit), so that w and b are loaded once per block, and the sums
// of dw / db stay in registers until a block's last row: one partial row per block goes to the workspace and a second kernel adds the partials in
// block order, so results do not depend on the order in which blocks run.  Sums and statistics are fp32; y / dx are rounded once.
// Loads and stores are 16 bytes at any alignment (the hardware splits what crosses a line), so an odd width costs only its last chunk.
// Measured: 108528 x 256 bf16 forward 20.3 us (5.5 TB/s), backward 29.1 (5.7) and 4 for the sums; 16384 x 4096 fp32 95 (5.6) and 158 (5.1), where a
// large copy reaches 5.1; 4099 x 1283 fp16 with a residual 14 and 26; 300 x 256 4.3.
#include "chunk.hpp"

namespace moy {

struct LnParams {
  const void* x; int64_t ldx;
  const void* r; int64_t ldr;
  const void* dy; int64_t ldd;
  const void* w; const void* b; int w_dtype;
  int64_t rows; int C; float eps;
  void* y; int64_t ldy;                    // forward: y; backward: dx
  float* mean; float* rstd;
  float* part;                             // backward: [gridDim.x][2][C] partial sums of dw, db (NULL: not wanted)
};

// The weights of a lane's chunk, in their own type (fp32, or the activations'): one branch for the chunk, so that its loads go out together.
template <typename T>
__device__ __forceinline__ void ln_weights(const void* p, int dtype, int c, int n, float dflt, float (&v)[Chunk<T>::VEC]) {
  constexpr int VEC = Chunk<T>::VEC;
  if (!p || n <= 0) {
#pragma unroll
    for (int e = 0; e < VEC; ++e) v[e] = dflt;
  } else if (dtype == DT<T>::code) {
    Chunk<T>::load(static_cast<const T*>(p) + c, n, v);
  } else {
    const float* f = static_cast<const float*>(p) + c;
    float lo[4], hi[4] = {0.f, 0.f, 0.f, 0.f};
    Chunk<float>::load(f, n, lo);
    if (n > 4) Chunk<float>::load(f + 4, n - 4, hi);
#pragma unroll
    for (int e = 0; e < VEC; ++e) v[e] = e < 4 ? lo[e] : hi[e & 3];
  }
}
// Sum over the TPR lanes (16, a wave, or the block) that hold one row; every lane gets it.  slots: LDS of one reduction round, not used again
// before another round's barrier has passed.
template <int TPR>
__device__ __forceinline__ float row_sum(float v, float* slots) {
  if constexpr (TPR == 16) {
    v += dpp_f<0xb1, 0xf>(0.f, v);          // quad sums
    v += dpp_f<0x4e, 0xf>(0.f, v);
    v += dpp_f<0x141, 0xf>(0.f, v);         // row_half_mirror: the other quad of eight lanes
    v += dpp_f<0x140, 0xf>(0.f, v);         // row_mirror: the other eight
    return v;
  } else {
    v = wave_sum(v);
    if constexpr (TPR > 64) {
      const int wave = threadIdx.x >> 6;
      if ((threadIdx.x & 63) == 0) slots[wave] = v;
      __syncthreads();
      v = 0.f;
#pragma unroll
      for (int k = 0; k < TPR / 64; ++k) v += slots[k];
    }
    return v;
  }
}

template <int TPR>
struct LnGeom {
  static constexpr int THREADS = TPR > 256 ? TPR : 256;
  static constexpr int GROUPS = THREADS / TPR;      // rows of a block at a time
  static constexpr int SLOTS = TPR > 64 ? TPR / 64 : 1;
};

template <typename T, int TPR, int NV>
__global__ __launch_bounds__(LnGeom<TPR>::THREADS) void ln_fwd_kernel(const LnParams p) {
  using G = LnGeom<TPR>;
  using K = Chunk<T>;
  constexpr int VEC = K::VEC;
  __shared__ float slots[2][G::SLOTS];
  const int t = threadIdx.x % TPR, group = threadIdx.x / TPR;
  float w[NV][VEC], b[NV][VEC];
  int left[NV];
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int c = (i * TPR + t) * VEC;
    left[i] = p.C - c;
    ln_weights<T>(p.w, p.w_dtype, c, left[i], 1.f, w[i]);
    ln_weights<T>(p.b, p.w_dtype, c, left[i], 0.f, b[i]);
  }
  for (int64_t row = (int64_t)blockIdx.x * G::GROUPS + group; row < p.rows; row += (int64_t)gridDim.x * G::GROUPS) {
    const T* x = static_cast<const T*>(p.x) + row * p.ldx;
    float v[NV][VEC];
    float s = 0.f;
#pragma unroll
    for (int i = 0; i < NV; ++i) K::load(x + (i * TPR + t) * VEC, left[i], v[i]);
    if (p.r) {
      const T* r = static_cast<const T*>(p.r) + row * p.ldr;
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        float u[VEC];
        K::load(r + (i * TPR + t) * VEC, left[i], u);
#pragma unroll
        for (int e = 0; e < VEC; ++e) v[i][e] += u[e];
      }
    }
#pragma unroll
    for (int i = 0; i < NV; ++i)
#pragma unroll
      for (int e = 0; e < VEC; ++e) s += v[i][e];
    const float mu = row_sum<TPR>(s, slots[0]) / (float)p.C;    // (a true quotient: a constant row comes out as exact zeros)
    float ss = 0.f;
#pragma unroll
    for (int i = 0; i < NV; ++i)
#pragma unroll
      for (int e = 0; e < VEC; ++e) {
        v[i][e] = e < left[i] ? v[i][e] - mu : 0.f;
        ss += v[i][e] * v[i][e];
      }
    const float rstd = 1.f / sqrtf(row_sum<TPR>(ss, slots[1]) / (float)p.C + p.eps);
    if (p.mean && t == 0) {
      p.mean[row] = mu;
      p.rstd[row] = rstd;
    }
    T* y = static_cast<T*>(p.y) + row * p.ldy;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
#pragma unroll
      for (int e = 0; e < VEC; ++e) v[i][e] = v[i][e] * rstd * w[i][e] + b[i][e];
      K::store(y + (i * TPR + t) * VEC, left[i], v[i]);
    }
  }
}

template <typename T, int TPR, int NV>
__global__ __launch_bounds__(LnGeom<TPR>::THREADS) void ln_bwd_kernel(const LnParams p) {
  using G = LnGeom<TPR>;
  using K = Chunk<T>;
  constexpr int VEC = K::VEC;
  __shared__ float slots[2][2][G::SLOTS];
  __shared__ float sums[TPR <= 64 ? G::GROUPS * TPR * VEC : 1];
  const int t = threadIdx.x % TPR, group = threadIdx.x / TPR;
  float w[NV][VEC], dw[NV][VEC], db[NV][VEC];
  int left[NV];
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int c = (i * TPR + t) * VEC;
    left[i] = p.C - c;
    ln_weights<T>(p.w, p.w_dtype, c, left[i], 1.f, w[i]);
#pragma unroll
    for (int e = 0; e < VEC; ++e) dw[i][e] = db[i][e] = 0.f;
  }
  const float inv = 1.f / (float)p.C;
  int turn = 0;
  for (int64_t row = (int64_t)blockIdx.x * G::GROUPS + group; row < p.rows; row += (int64_t)gridDim.x * G::GROUPS, turn ^= 1) {
    const T* x = static_cast<const T*>(p.x) + row * p.ldx;
    const T* dy = static_cast<const T*>(p.dy) + row * p.ldd;
    const float mu = p.mean[row], rstd = p.rstd[row];
    float v[NV][VEC], g[NV][VEC];
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      K::load(x + (i * TPR + t) * VEC, left[i], v[i]);
      K::load(dy + (i * TPR + t) * VEC, left[i], g[i]);
    }
    if (p.r) {
      const T* r = static_cast<const T*>(p.r) + row * p.ldr;
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        float u[VEC];
        K::load(r + (i * TPR + t) * VEC, left[i], u);
#pragma unroll
        for (int e = 0; e < VEC; ++e) v[i][e] += u[e];
      }
    }
    float a = 0.f, c = 0.f;
#pragma unroll
    for (int i = 0; i < NV; ++i)
#pragma unroll
      for (int e = 0; e < VEC; ++e) {        // past the row's end g is 0, so what v holds there does not count
        v[i][e] = (v[i][e] - mu) * rstd;
        dw[i][e] += g[i][e] * v[i][e];
        db[i][e] += g[i][e];
        g[i][e] *= w[i][e];
        a += g[i][e];
        c += g[i][e] * v[i][e];
      }
    if (p.y) {
      a = row_sum<TPR>(a, slots[turn][0]) * inv;
      c = row_sum<TPR>(c, slots[turn][1]) * inv;
      T* dx = static_cast<T*>(p.y) + row * p.ldy;
#pragma unroll
      for (int i = 0; i < NV; ++i) {
#pragma unroll
        for (int e = 0; e < VEC; ++e) g[i][e] = (g[i][e] - a - v[i][e] * c) * rstd;
        K::store(dx + (i * TPR + t) * VEC, left[i], g[i]);
      }
    }
  }
  if (!p.part) return;
  float* part = p.part + (int64_t)blockIdx.x * 2 * p.C;
#pragma unroll
  for (int k = 0; k < 2; ++k)
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      float (&d)[VEC] = k ? db[i] : dw[i];
      const int c = (i * TPR + t) * VEC;
      if constexpr (G::GROUPS > 1) {         // the block's groups hold the same columns: add them in group order
        __syncthreads();
#pragma unroll
        for (int e = 0; e < VEC; ++e) sums[(group * VEC + e) * TPR + t] = d[e];
        __syncthreads();
        for (int s = threadIdx.x; s < TPR * VEC; s += G::THREADS) {
          const int e = s % VEC, tt = s / VEC, col = (i * TPR + tt) * VEC + e;
          float sum = 0.f;
#pragma unroll
          for (int gg = 0; gg < G::GROUPS; ++gg) sum += sums[(gg * VEC + e) * TPR + tt];
          if (col < p.C) part[k * p.C + col] = sum;
        }
      } else {
#pragma unroll
        for (int e = 0; e < VEC; ++e)
          if (e < left[i]) part[k * p.C + c + e] = d[e];
      }
    }
}

// Lanes and chunks for a row of `chunks` 16-byte pieces: the fewest lanes that hold it in one or two chunks each, 2048 chunks at most (16384 channels of 16
// bits, 8192 of fp32).  The forward has the registers for three chunks in a wave's lanes, which save it the block's barriers; the backward has not (65536 x 1536
// bf16 with three chunks against a block of 256 lanes: forward 74 us / 108, backward 171 / 149; with four, 65536 x 2048: 134 / 116).
static int ln_lanes(int chunks, bool bwd) {
  return chunks <= 32 ? 16 : chunks <= (bwd ? 128 : 192) ? 64 : chunks <= 512 ? 256 : chunks <= 2048 ? 1024 : 0;
}

static int ln_chunks(int C, int dtype) { return dtype == MOY_F32 ? (C + 3) / 4 : (C + 7) / 8; }

// Blocks that walk the rows: four of 256 threads to a compute unit, two of 1024.
static int ln_blocks(int64_t rows, int lanes) {
  const int64_t groups = lanes > 256 ? 1 : 256 / lanes, want = (rows + groups - 1) / groups, most = lanes > 256 ? 512 : 1024;
  return (int)(want < most ? want : most);
}

template <typename T, bool BWD>
static int ln_launch(const LnParams& p, int lanes, int chunks, int blocks, hipStream_t st) {
#define MOY_LN(TPR, NV)                                                                                                        \
  {                                                                                                                            \
    if constexpr (BWD) hipLaunchKernelGGL((ln_bwd_kernel<T, TPR, NV>), dim3(blocks), dim3(LnGeom<TPR>::THREADS), 0, st, p);      \
    else hipLaunchKernelGGL((ln_fwd_kernel<T, TPR, NV>), dim3(blocks), dim3(LnGeom<TPR>::THREADS), 0, st, p);                   \
    return launch_status();                                                                                                    \
  }
  const bool one = chunks <= lanes;
  switch (lanes) {
    case 16: if (one) MOY_LN(16, 1) else MOY_LN(16, 2)
    case 64:
      if constexpr (!BWD) {
        if (chunks > 128) MOY_LN(64, 3)
      }
      if (one) MOY_LN(64, 1) else MOY_LN(64, 2)
    case 256: if (one) MOY_LN(256, 1) else MOY_LN(256, 2)
    default: if (one) MOY_LN(1024, 1) else MOY_LN(1024, 2)
  }
#undef MOY_LN
}

template <bool BWD>
static int ln_dispatch(const LnParams& p, int dtype, hipStream_t st) {
  const int chunks = ln_chunks(p.C, dtype), lanes = ln_lanes(chunks, BWD);
  const int blocks = ln_blocks(p.rows, lanes);
  switch (dtype) {
    case MOY_F32: return ln_launch<float, BWD>(p, lanes, chunks, blocks, st);
    case MOY_BF16: return ln_launch<bf16_t, BWD>(p, lanes, chunks, blocks, st);
    default: return ln_launch<f16_t, BWD>(p, lanes, chunks, blocks, st);
  }
}

static int ln_check(int64_t rows, int C, int dtype, int w_dtype, bool weights) {
  if (rows <= 0 || C <= 0 || dtype < MOY_F32 || dtype > MOY_F16) return MOY_EINVAL;
  if (weights && w_dtype != MOY_F32 && w_dtype != dtype) return MOY_EINVAL;
  return ln_lanes(ln_chunks(C, dtype), true) ? MOY_OK : MOY_ENOSYS;
}

}  // namespace moy

using namespace moy;

extern "C" int moy_layer_norm(const void* x, int64_t ldx, const void* r, int64_t ldr, const void* w, const void* b, int w_dtype, int64_t rows, int C,
                              float eps, void* y, int64_t ldy, float* mean, float* rstd, int dtype, void* stream) {
  const int rc = ln_check(rows, C, dtype, w_dtype, w || b);
  if (rc != MOY_OK) return rc;
  if (!x || !y || (mean == nullptr) != (rstd == nullptr) || !(eps >= 0.f)) return MOY_EINVAL;
  if (rows > 1 && (ldx < 0 || ldy < C || (r && ldr < 0))) return MOY_EINVAL;
  if (!aligned_as(x, dtype) || !aligned_as(y, dtype) || !aligned_as(r, dtype) || !aligned_as(w, w_dtype) || !aligned_as(b, w_dtype)) return MOY_EINVAL;
  LnParams p{};
  p.x = x; p.ldx = ldx; p.r = r; p.ldr = ldr; p.w = w; p.b = b; p.w_dtype = w_dtype;
  p.rows = rows; p.C = C; p.eps = eps; p.y = y; p.ldy = ldy; p.mean = mean; p.rstd = rstd;
  return ln_dispatch<false>(p, dtype, static_cast<hipStream_t>(stream));
}

extern "C" int64_t moy_layer_norm_bwd_ws(int64_t rows, int C, int dtype) {
  const int rc = ln_check(rows, C, dtype, MOY_F32, false);
  if (rc != MOY_OK) return rc;
  return (int64_t)ln_blocks(rows, ln_lanes(ln_chunks(C, dtype), true)) * 2 * C;
}

extern "C" int moy_layer_norm_bwd(const void* dy, int64_t ldd, const void* x, int64_t ldx, const void* r, int64_t ldr, const void* w, int w_dtype,
                                  const float* mean, const float* rstd, int64_t rows, int C, void* dx, int64_t ldo, void* dw, void* db, float* ws,
                                  int64_t ws_len, int dtype, void* stream) {
  const int rc = ln_check(rows, C, dtype, w_dtype, w || dw || db);
  if (rc != MOY_OK) return rc;
  if (!dy || !x || !mean || !rstd || (!dx && !dw && !db)) return MOY_EINVAL;
  if (rows > 1 && (ldd < 0 || ldx < 0 || (r && ldr < 0) || (dx && ldo < C))) return MOY_EINVAL;
  if (!aligned_as(dy, dtype) || !aligned_as(x, dtype) || !aligned_as(r, dtype) || !aligned_as(dx, dtype) || !aligned_as(w, w_dtype) ||
      !aligned_as(dw, w_dtype) || !aligned_as(db, w_dtype))
    return MOY_EINVAL;
  const bool sums = dw || db;
  const int blocks = ln_blocks(rows, ln_lanes(ln_chunks(C, dtype), true));
  if (sums && (!ws || ws_len < (int64_t)blocks * 2 * C)) return MOY_EINVAL;
  LnParams p{};
  p.x = x; p.ldx = ldx; p.r = r; p.ldr = ldr; p.dy = dy; p.ldd = ldd; p.w = w; p.w_dtype = w_dtype;
  p.rows = rows; p.C = C; p.y = dx; p.ldy = ldo; p.mean = const_cast<float*>(mean); p.rstd = const_cast<float*>(rstd);
  p.part = sums ? ws : nullptr;
  hipStream_t st = static_cast<hipStream_t>(stream);
  const int k = ln_dispatch<true>(p, dtype, st);
  if (k != MOY_OK || !sums) return k;
  hipLaunchKernelGGL(column_sums_kernel, dim3((2 * C + 31) / 32), dim3(1024), 0, st, ws, blocks, C, C, dw, db, w_dtype);
  return launch_status();
}
