// Residual addition with root-mean-square norm, rows of D elements:
//
//   h = x + r  (float32, rounded once to r's type; h = x without a residual)
//   rstd = 1 / sqrt(mean_j h_j^2 + eps),   y = (h rstd) w
//
// or, with the output in 8 bits, q = e4m3(y 448 / amax), scale = amax / 448
// with amax the row's largest |y| (at least 2^-100: a row of zeros has a finite
// scale).  The norm is taken of the stored h, so that the backward recomputes
// it from what the forward left.  With g = dy w:
//
//   dh = dh_out + rstd (g - n mean_j(g_j n_j)),  n = h rstd;   dx = dr = dh;   dw = sum over rows of dy n
//
// Every kernel is bound by the bytes it moves: one read of x and r (dy, dh_out
// and h in the backward), one write of h and y (dx, dr).  A row stays in
// registers between its reduction and its output, so nothing is read twice
// (past 32768 elements, 16384 in the backward, a row is read again, through the
// cache).
//
// Measured (MI355X): 32768 x 768, float32 stream and bf16 branch, 138 us
// forward and backward, 5.1 TB/s; 8191 x 8192 in bf16 with rows in 8 bits 84 to
// 87 us, 5.4 TB/s (a large copy reaches 4.9 to 5.5); 32 x 8192 2.8 us in a captured
// loop, three loads of memory latency one after another.
//
// Threads per row: eight to 1024, a run of 8 elements each to 8192 elements
// (norm_shape); up to one wave there is no barrier at all.
//
// The backward's workgroups walk over rows in a stride of the grid and keep
// their columns' part of dw in registers; the parts are added in workgroup
// order by a second launch, so that dw has the same bits on every run.
#include "nsa_launch.h"
#include "nsa_rows.h"

namespace nsa {

constexpr float kQ8Max = 448.0f;            // largest e4m3 value
constexpr float kQ8Floor = 0x1p-100f;
constexpr int kNormRegMax = 32768;           // widest row held in registers (forward)
constexpr int kNormBwdMax = 16384;           // ... and with its gradient and its part of dw (backward)
constexpr int kNormMax = 1 << 24;            // widest row
constexpr int64_t kNormSlice = 1 << 21;      // rows of one launch

struct NormArgs {
  const void *x, *res, *w;
  void *h, *y;
  float *scale, *rstd;
  int64_t rows;
  int D;
  float eps, inv_d;
  bool w_bf16, y_bf16;
};

__device__ __forceinline__ uint32_t abs_bits(float x) { return __float_as_uint(x) & 0x7fffffffu; }

// 8 floats as e4m3 (round to nearest even; |v| <= 448 but for NaN)
__device__ __forceinline__ void store_q8(uint8_t* p, int n, const float (&f)[8]) {
  typedef uint32_t u32x2u __attribute__((ext_vector_type(2), aligned(1)));
  int a = __builtin_amdgcn_cvt_pk_fp8_f32(f[0], f[1], 0, false);
  a = __builtin_amdgcn_cvt_pk_fp8_f32(f[2], f[3], a, true);
  int b = __builtin_amdgcn_cvt_pk_fp8_f32(f[4], f[5], 0, false);
  b = __builtin_amdgcn_cvt_pk_fp8_f32(f[6], f[7], b, true);
  if (n >= 8) {
    *reinterpret_cast<u32x2u*>(p) = (u32x2u){(uint32_t)a, (uint32_t)b};
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j)
      if (j < n) p[j] = (uint8_t)((uint32_t)(j < 4 ? a : b) >> (8 * (j & 3)));
  }
}

// h of one run: x + r rounded to r's type (RES), or x itself
template <typename XT, typename RT, bool RES>
__device__ __forceinline__ void norm_sum8(const NormArgs& a, int64_t at, int n, float (&h)[8]) {
  load_run8(static_cast<const XT*>(a.x) + at, n, h);
  if (RES) {
    float r[8];
    load_run8(static_cast<const RT*>(a.res) + at, n, r);
#pragma unroll
    for (int j = 0; j < 8; ++j) h[j] = (float)(RT)(h[j] + r[j]);
  }
}

// TPR threads a row, NV runs of 8 a thread (NV = 0: any length, h formed again for every pass).
template <typename XT, typename RT, bool RES, bool Q8, int TPR, int NV>
__global__ __launch_bounds__(TPR <= 64 ? 256 : TPR) void k_norm_fwd(const NormArgs a) {
  constexpr int W = TPR > kWave ? TPR / kWave : 1;
  __shared__ float red[2][W];
  __shared__ uint32_t redm[W];
  const int t = threadIdx.x & (TPR - 1);
  const int64_t row = TPR <= 64 ? (int64_t)blockIdx.x * (256 / TPR) + threadIdx.x / TPR : (int64_t)blockIdx.x;
  if (TPR <= 64 && row >= a.rows) return;   // (all of a row's lanes; no barrier follows for these)
  const int D = a.D;
  const int64_t base = row * D;
  const int nrun = NV > 0 ? NV : (D + 8 * TPR - 1) / (8 * TPR);
  float h[NV > 0 ? NV : 1][8];
  float ss = 0.0f;
#pragma unroll
  for (int i = 0; i < nrun; ++i) {
    float(&hi)[8] = h[NV > 0 ? i : 0];
    const int c = 8 * (i * TPR + t), n = D - c;
    norm_sum8<XT, RT, RES>(a, base + c, n, hi);
#pragma unroll
    for (int j = 0; j < 8; ++j) ss += hi[j] * hi[j];
    if (RES && n > 0) store_run8(static_cast<RT*>(a.h) + base + c, n, hi);
  }
  ss = row_sum<TPR>(ss, red[0]);
  const float rstd = 1.0f / sqrtf(ss * a.inv_d + a.eps);
  if (a.rstd != nullptr && t == 0) a.rstd[row] = rstd;
  uint32_t am = 0;   // |y| as bits: the order of the magnitudes, NaN above infinity
#pragma unroll
  for (int i = 0; i < nrun; ++i) {
    float(&hi)[8] = h[NV > 0 ? i : 0];
    const int c = 8 * (i * TPR + t), n = D - c;
    if (NV == 0) norm_sum8<XT, RT, RES>(a, base + c, n, hi);
    float wv[8];
    load_run8_of(a.w, a.w_bf16, c, n, wv);
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      hi[j] = (hi[j] * rstd) * wv[j];
      if (Q8 && j < n) am = max(am, abs_bits(hi[j]));
    }
    if (!Q8 && n > 0) {
      if (a.y_bf16)
        store_run8(static_cast<bf16*>(a.y) + base + c, n, hi);
      else
        store_run8(static_cast<float*>(a.y) + base + c, n, hi);
    }
  }
  if (Q8) {
    // (a non-negative float's bits have its order, NaN's above infinity's)
    am = lanes_all<(TPR < kWave ? TPR : kWave)>(am, [](uint32_t x, uint32_t y) { return x > y ? x : y; });
    if (W > 1) {
      if ((threadIdx.x & (kWave - 1)) == 0) redm[threadIdx.x / kWave] = am;
      __syncthreads();
#pragma unroll
      for (int i = 0; i < W; ++i) am = max(am, redm[i]);
    }
    const float amax = __uint_as_float(max(am, __float_as_uint(kQ8Floor)));
    const float inv = kQ8Max / amax;
    if (t == 0) a.scale[row] = amax / kQ8Max;
#pragma unroll
    for (int i = 0; i < nrun; ++i) {
      float(&hi)[8] = h[NV > 0 ? i : 0];
      const int c = 8 * (i * TPR + t), n = D - c;
      if (NV == 0) {
        norm_sum8<XT, RT, RES>(a, base + c, n, hi);
        float wv[8];
        load_run8_of(a.w, a.w_bf16, c, n, wv);
#pragma unroll
        for (int j = 0; j < 8; ++j) hi[j] = (hi[j] * rstd) * wv[j];
      }
#pragma unroll
      for (int j = 0; j < 8; ++j) hi[j] *= inv;
      if (n > 0) store_q8(static_cast<uint8_t*>(a.y) + base + c, n, hi);
    }
  }
}

struct NormBwdArgs {
  const void *dy, *dh, *h, *w;
  const float* rstd;
  void *dx, *dres;
  float* part;            // [gridDim.x][D], or null
  int64_t rows;
  int D;
  float inv_d;
  bool w_bf16, dx_bf16;
};

// YT: dy; RT: h, dh and dres.  dres is null where dx serves both (one type).
template <typename YT, typename RT, int TPR, int NV>
__global__ __launch_bounds__(TPR <= 64 ? 256 : TPR) void k_norm_bwd(const NormBwdArgs a) {
  constexpr int W = TPR > kWave ? TPR / kWave : 1;
  constexpr int RPG = TPR <= 64 ? 256 / TPR : 1;   // rows at a time
  __shared__ float red[2][W];
  __shared__ float dws[RPG > 1 ? 8 * TPR * NV : 1];
  const int t = threadIdx.x & (TPR - 1);
  const int sub = threadIdx.x / TPR;
  const int D = a.D;
  // where the registers hold them: the weights for all rows, and dh asked for with the rest of a row
  constexpr bool kHold = NV * TPR <= 1024;
  float w[kHold ? NV : 1][8], dw[NV][8];
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    if (kHold) load_run8_of(a.w, a.w_bf16, 8 * (i * TPR + t), D - 8 * (i * TPR + t), w[kHold ? i : 0]);
#pragma unroll
    for (int j = 0; j < 8; ++j) dw[i][j] = 0.0f;
  }
  int turn = 0;
  for (int64_t row = (int64_t)blockIdx.x * RPG + sub; row < a.rows; row += (int64_t)gridDim.x * RPG) {
    const int64_t base = row * D;
    const float rstd = a.rstd[row];
    float n_[NV][8], g[NV][8], d[kHold ? NV : 1][8];
    float dot = 0.0f;
    auto load_dh = [&](int i, float(&v)[8]) {
      const int c = 8 * (i * TPR + t);
      if (a.dh != nullptr) {
        load_run8(static_cast<const RT*>(a.dh) + base + c, D - c, v);
      } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] = 0.0f;
      }
    };
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int c = 8 * (i * TPR + t), n = D - c;
      load_run8(static_cast<const RT*>(a.h) + base + c, n, n_[i]);
      load_run8(static_cast<const YT*>(a.dy) + base + c, n, g[i]);
      if (kHold) load_dh(i, d[i]);
    }
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      float(&wi)[8] = w[kHold ? i : 0];
      if (!kHold) load_run8_of(a.w, a.w_bf16, 8 * (i * TPR + t), D - 8 * (i * TPR + t), wi);
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        n_[i][j] *= rstd;
        dw[i][j] += g[i][j] * n_[i][j];
        g[i][j] *= wi[j];
        dot += g[i][j] * n_[i][j];
      }
    }
    // two buffers in turn: the next row's sum is not written over one still being read
    dot = row_sum<TPR>(dot, red[turn & 1]) * a.inv_d;
    ++turn;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int c = 8 * (i * TPR + t), n = D - c;
      float(&di)[8] = d[kHold ? i : 0];
      if (!kHold) load_dh(i, di);
#pragma unroll
      for (int j = 0; j < 8; ++j) di[j] += rstd * (g[i][j] - n_[i][j] * dot);
      if (n > 0) {
        if (a.dx_bf16)
          store_run8(static_cast<bf16*>(a.dx) + base + c, n, di);
        else
          store_run8(static_cast<float*>(a.dx) + base + c, n, di);
        if (a.dres != nullptr) store_run8(static_cast<RT*>(a.dres) + base + c, n, di);
      }
    }
  }
  if (a.part == nullptr) return;
  float* out = a.part + (int64_t)blockIdx.x * D;
  if constexpr (RPG == 1) {
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int c = 8 * (i * TPR + t);
      if (c < D) store_run8(out + c, D - c, dw[i]);
    }
  } else {
    static_assert(NV == 1, "a row of at most a wave is one run a lane");
    // the rows of a wave by halves, then the waves' parts in wave order
#pragma unroll
    for (int x = TPR; x < kWave; x <<= 1)
#pragma unroll
      for (int j = 0; j < 8; ++j) dw[0][j] += __shfl_xor(dw[0][j], x, kWave);
    const int w = threadIdx.x / kWave;
    for (int s = 0; s < 4; ++s) {
      if (w == s && (threadIdx.x & (kWave - 1)) < TPR) {
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const int c = 8 * t + j;
          if (c < D) dws[c] = s == 0 ? dw[0][j] : dws[c] + dw[0][j];
        }
      }
      __syncthreads();
    }
    for (int c = threadIdx.x; c < D; c += 256) out[c] = dws[c];
  }
}

// Rows past kNormBwdMax: one workgroup a row, read twice.
template <typename YT, typename RT>
__global__ __launch_bounds__(1024) void k_norm_bwd_long(const NormBwdArgs a) {
  __shared__ float red[2][16];
  const int D = a.D;
  int turn = 0;
  for (int64_t row = blockIdx.x; row < a.rows; row += gridDim.x, ++turn) {
    const int64_t base = row * D;
    const float rstd = a.rstd[row];
    float dot = 0.0f;
    for (int c = 8 * threadIdx.x; c < D; c += 8 * 1024) {
      float h[8], g[8], w[8];
      load_run8(static_cast<const RT*>(a.h) + base + c, D - c, h);
      load_run8(static_cast<const YT*>(a.dy) + base + c, D - c, g);
      load_run8_of(a.w, a.w_bf16, c, D - c, w);
#pragma unroll
      for (int j = 0; j < 8; ++j) dot += g[j] * w[j] * (h[j] * rstd);
    }
    dot = row_sum<1024>(dot, red[turn & 1]) * a.inv_d;
    for (int c = 8 * threadIdx.x; c < D; c += 8 * 1024) {
      const int n = D - c;
      float h[8], g[8], w[8], d[8] = {0, 0, 0, 0, 0, 0, 0, 0};
      load_run8(static_cast<const RT*>(a.h) + base + c, n, h);
      load_run8(static_cast<const YT*>(a.dy) + base + c, n, g);
      load_run8_of(a.w, a.w_bf16, c, n, w);
      if (a.dh != nullptr) load_run8(static_cast<const RT*>(a.dh) + base + c, n, d);
#pragma unroll
      for (int j = 0; j < 8; ++j) d[j] += rstd * (g[j] * w[j] - h[j] * rstd * dot);
      if (a.dx_bf16)
        store_run8(static_cast<bf16*>(a.dx) + base + c, n, d);
      else
        store_run8(static_cast<float*>(a.dx) + base + c, n, d);
      if (a.dres != nullptr) store_run8(static_cast<RT*>(a.dres) + base + c, n, d);
    }
  }
}

// Parts of dw for such rows: 2048 columns and every gridDim.y-th row a workgroup.
template <typename YT, typename RT>
__global__ __launch_bounds__(256) void k_norm_dw_wide(const NormBwdArgs a) {
  const int c = 8 * ((int)blockIdx.x * 256 + (int)threadIdx.x), n = a.D - c;
  if (n <= 0) return;
  float dw[8] = {0, 0, 0, 0, 0, 0, 0, 0};
#pragma unroll 2
  for (int64_t row = blockIdx.y; row < a.rows; row += gridDim.y) {
    float h[8], g[8];
    load_run8(static_cast<const RT*>(a.h) + row * a.D + c, n, h);
    load_run8(static_cast<const YT*>(a.dy) + row * a.D + c, n, g);
    const float rstd = a.rstd[row];
#pragma unroll
    for (int j = 0; j < 8; ++j) dw[j] += g[j] * (h[j] * rstd);
  }
  store_run8(a.part + (int64_t)blockIdx.y * a.D + c, n, dw);
}

// dw[c] = sum of part[p][c]: 16 columns a workgroup (64-byte pieces of a part), 64
// interleaved sums over the parts, added in order.
__global__ __launch_bounds__(1024) void k_norm_dw(const float* __restrict__ part, int nparts, int D, void* dw,
                                                  bool w_bf16) {
  __shared__ float acc[64][17];
  const int x = threadIdx.x & 15, s = threadIdx.x >> 4;
  const int c = blockIdx.x * 16 + x;
  float v = 0.0f;
  if (c < D) {
#pragma unroll 8
    for (int p = s; p < nparts; p += 64) v += part[(int64_t)p * D + c];
  }
  acc[s][x] = v;
  __syncthreads();
  if (s < 4) {   // 16 sums each by the first wave, then those four
    float t = 0.0f;
#pragma unroll
    for (int i = 0; i < 16; ++i) t += acc[16 * s + i][x];
    t += __shfl_xor(t, 16, kWave);
    t += __shfl_xor(t, 32, kWave);
    if (s == 0 && c < D) {
      if (w_bf16)
        static_cast<bf16*>(dw)[c] = (bf16)t;
      else
        static_cast<float*>(dw)[c] = t;
    }
  }
}

// Threads a row and runs a thread: the fewest threads that hold the row with one
// run each (8191 x 8192 in bf16 with rows in 8 bits: 84 us with 1024 threads, 95
// with four runs in 256; 32768 x 768 forward and backward, float32 stream: 138 us
// with 128 threads, 142 with two runs in 64); past 8192 elements two or four runs in 1024.
struct NormShape {
  int tpr, nv;
};
#define NSA_NORM_SHAPES(X) X(8, 1) X(16, 1) X(32, 1) X(64, 1) X(128, 1) X(256, 1) X(512, 1) X(1024, 1) X(1024, 2)
static NormShape norm_shape(int D) {
  const int runs = (D + 7) / 8;
#define NSA_NORM_FITS(TPR, NV) \
  if (runs <= TPR * NV) return {TPR, NV};
  NSA_NORM_SHAPES(NSA_NORM_FITS)
#undef NSA_NORM_FITS
  return {1024, D <= kNormRegMax ? 4 : 0};
}

template <typename XT, typename RT, bool RES, bool Q8>
static int norm_fwd_launch(const NormArgs& a, hipStream_t s) {
  const NormShape sh = norm_shape(a.D);
#define NSA_NORM_CASE(TPR, NV)                                                                    \
  if (sh.tpr == TPR && sh.nv == NV) {                                                             \
    const int64_t grid = TPR <= 64 ? (a.rows + 256 / TPR - 1) / (256 / TPR) : a.rows;             \
    k_norm_fwd<XT, RT, RES, Q8, TPR, NV><<<(unsigned)grid, TPR <= 64 ? 256 : TPR, 0, s>>>(a);     \
    return nsa_launch_status();                                                                   \
  }
  NSA_NORM_SHAPES(NSA_NORM_CASE) NSA_NORM_CASE(1024, 4) NSA_NORM_CASE(1024, 0)
#undef NSA_NORM_CASE
  return NSA_ERR_SHAPE;
}

template <typename XT, typename RT>
static int norm_fwd_as(const NormArgs& a, bool q8, hipStream_t s) {
  if (a.res != nullptr) return q8 ? norm_fwd_launch<XT, RT, true, true>(a, s) : norm_fwd_launch<XT, RT, true, false>(a, s);
  if constexpr (sizeof(XT) == sizeof(RT))
    return q8 ? norm_fwd_launch<XT, RT, false, true>(a, s) : norm_fwd_launch<XT, RT, false, false>(a, s);
  return NSA_ERR_DTYPE;
}

// Parts of dw: a workgroup of the backward each, eight to a compute unit or what
// its waves hold; past kNormBwdMax a row group of k_norm_dw_wide.
static int64_t norm_bwd_groups(int64_t rows, int D, int cu) {
  if (D > kNormBwdMax) return rows < 128 ? rows : 128;
  const NormShape sh = norm_shape(D);
  const int rpg = sh.tpr <= 64 ? 256 / sh.tpr : 1;
  const int64_t groups = (rows + rpg - 1) / rpg;
  const int64_t most = (int64_t)cu * (sh.tpr <= 256 ? 8 : 2048 / sh.tpr);
  return groups < most ? groups : most;
}

template <typename YT, typename RT>
static int norm_bwd_launch(NormBwdArgs a, void* dw, hipStream_t s) {
  const int cu = device_cu_count(s);
  const NormShape sh = norm_shape(a.D);
  const int64_t grid = norm_bwd_groups(a.rows, a.D, cu);
  bool done = false;
  if (a.D > kNormBwdMax) {
    k_norm_bwd_long<YT, RT><<<(unsigned)(a.rows < 8192 ? a.rows : 8192), 1024, 0, s>>>(a);
    if (dw != nullptr)
      k_norm_dw_wide<YT, RT><<<dim3((unsigned)((a.D + 2047) / 2048), (unsigned)grid), 256, 0, s>>>(a);
    done = true;
  }
#define NSA_NORM_CASE(TPR, NV)                                                            \
  if (!done && sh.tpr == TPR && sh.nv == NV) {                                            \
    k_norm_bwd<YT, RT, TPR, NV><<<(unsigned)grid, TPR <= 64 ? 256 : TPR, 0, s>>>(a);      \
    done = true;                                                                          \
  }
  NSA_NORM_SHAPES(NSA_NORM_CASE)
#undef NSA_NORM_CASE
  if (!done) return NSA_ERR_SHAPE;
  if (dw != nullptr)
    k_norm_dw<<<(unsigned)((a.D + 15) / 16), 1024, 0, s>>>(a.part, (int)grid, a.D, dw, a.w_bf16);
  return nsa_launch_status();
}

static bool norm_type(int dtype) { return dtype == NSA_F32 || dtype == NSA_BF16; }

}  // namespace nsa

extern "C" int nsa_norm_fwd(const void* x, const void* res, const void* w, void* h, void* y, float* scale,
                            float* rstd, int64_t rows, int D, float eps, int x_dtype, int h_dtype, int w_dtype,
                            int y_dtype, void* stream) {
  using namespace nsa;
  NSA_CHECK(rows >= 0 && rows <= 0x7fffffffLL && D >= 1 && D <= kNormMax, NSA_ERR_SHAPE);
  NSA_CHECK(norm_type(x_dtype) && norm_type(h_dtype) && norm_type(w_dtype), NSA_ERR_DTYPE);
  NSA_CHECK(norm_type(y_dtype) || y_dtype == NSA_E4M3, NSA_ERR_DTYPE);
  NSA_CHECK(res != nullptr || x_dtype == h_dtype, NSA_ERR_DTYPE);
  if (rows == 0) return NSA_OK;
  NSA_CHECK(x != nullptr && w != nullptr && y != nullptr, NSA_ERR_ARG);
  NSA_CHECK(res == nullptr || h != nullptr, NSA_ERR_ARG);
  NSA_CHECK(y_dtype != NSA_E4M3 || scale != nullptr, NSA_ERR_ARG);
  const hipStream_t s = static_cast<hipStream_t>(stream);
  const bool q8 = y_dtype == NSA_E4M3;
  const size_t xs = x_dtype == NSA_BF16 ? 2 : 4, hs = h_dtype == NSA_BF16 ? 2 : 4;
  const size_t ys = q8 ? 1 : y_dtype == NSA_BF16 ? 2 : 4;
  // 2^21 rows a launch: a grid holds less than 2^32 threads
  for (int64_t r0 = 0; r0 < rows; r0 += kNormSlice) {
    const int64_t n = rows - r0 < kNormSlice ? rows - r0 : kNormSlice, at = r0 * D;
    const NormArgs a{static_cast<const char*>(x) + at * xs,
                     res == nullptr ? nullptr : static_cast<const char*>(res) + at * hs,
                     w,
                     h == nullptr ? nullptr : static_cast<char*>(h) + at * hs,
                     static_cast<char*>(y) + at * ys,
                     scale == nullptr ? nullptr : scale + r0,
                     rstd == nullptr ? nullptr : rstd + r0,
                     n, D, eps, 1.0f / (float)D, w_dtype == NSA_BF16, y_dtype == NSA_BF16};
    int rc;
    if (x_dtype == NSA_BF16)
      rc = h_dtype == NSA_BF16 ? norm_fwd_as<bf16, bf16>(a, q8, s) : norm_fwd_as<bf16, float>(a, q8, s);
    else
      rc = h_dtype == NSA_BF16 ? norm_fwd_as<float, bf16>(a, q8, s) : norm_fwd_as<float, float>(a, q8, s);
    if (rc != NSA_OK) return rc;
  }
  return NSA_OK;
}

extern "C" size_t nsa_norm_bwd_workspace(int64_t rows, int D, void* stream) {
  using namespace nsa;
  if (rows < 0 || rows > 0x7fffffffLL || D < 1 || D > kNormMax) return 0;
  if (rows == 0) return 16;
  return (size_t)norm_bwd_groups(rows, D, device_cu_count(static_cast<hipStream_t>(stream))) * D * sizeof(float);
}

extern "C" int nsa_norm_bwd(const void* dy, const void* dh, const void* h, const void* w, const float* rstd, void* dx,
                            void* dres, void* dw, void* workspace, size_t workspace_bytes, int64_t rows, int D,
                            int x_dtype, int h_dtype, int w_dtype, int y_dtype, void* stream) {
  using namespace nsa;
  NSA_CHECK(rows >= 1 && rows <= 0x7fffffffLL && D >= 1 && D <= kNormMax, NSA_ERR_SHAPE);
  NSA_CHECK(norm_type(x_dtype) && norm_type(h_dtype) && norm_type(w_dtype) && norm_type(y_dtype), NSA_ERR_DTYPE);
  NSA_CHECK(dy != nullptr && h != nullptr && w != nullptr && rstd != nullptr && dx != nullptr, NSA_ERR_ARG);
  const hipStream_t s = static_cast<hipStream_t>(stream);
  float* part = nullptr;
  if (dw != nullptr) {
    NSA_CHECK(workspace != nullptr && workspace_bytes >= nsa_norm_bwd_workspace(rows, D, stream), NSA_ERR_WORKSPACE);
    part = static_cast<float*>(workspace);
  }
  const NormBwdArgs a{dy, dh, h, w, rstd, dx, dres, part, rows, D, 1.0f / (float)D, w_dtype == NSA_BF16,
                      x_dtype == NSA_BF16};
  if (y_dtype == NSA_BF16)
    return h_dtype == NSA_BF16 ? norm_bwd_launch<bf16, bf16>(a, dw, s) : norm_bwd_launch<bf16, float>(a, dw, s);
  return h_dtype == NSA_BF16 ? norm_bwd_launch<float, bf16>(a, dw, s) : norm_bwd_launch<float, float>(a, dw, s);
}
