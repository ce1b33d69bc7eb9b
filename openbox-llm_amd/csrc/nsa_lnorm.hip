// Residual addition with layer norm, rows of D elements:
//
//   h = x + r  (float32, rounded once to r's type; h = x without a residual)
//   mu = mean_j h_j,  rstd = 1 / sqrt(mean_j (h_j - mu)^2 + eps),  n = (h - mu) rstd,  y = n w + b
//
// The norm is taken of the stored h, so that the backward recomputes it from what
// the forward left.  With g = dy w:
//
//   dh = dh_out + rstd (g - mean_j g_j - n mean_j(g_j n_j));   dx = dr = dh
//   dw = sum over rows of dy n,   db = sum over rows of dy
//
// The mean is summed in 64 bits and rounded once: a sum in 32, or its product with a
// rounded 1 / D, is off by steps of the elements' size, which rows far off zero show
// beside their deviation (41 times 16384 came out as 0.19, not 0).
//
// Every kernel is bound by the bytes it moves: one read of x and r (dy, dh_out and
// h in the backward), one write of h and y (dx, dr).  A row stays in registers, so
// that the squares are taken about the mean itself (a sum of squares less the
// squared mean loses the variance of rows far off zero); past 32768 elements, 16384
// in the backward, a row is read again, through the cache.
//
// Threads per row: eight to 1024, a run of 8 elements each to 8192 elements
// (ln_shape); up to one wave there is no barrier at all.
//
// The backward's workgroups walk over rows in a stride of the grid and keep their
// columns' parts of dw and db in registers; the parts are added in workgroup order
// by a second launch, so that both have the same bits on every run.
//
// Measured, against a copy's 5.4 TB/s: 32768 x 768 (bf16 branch, float32 stream) 60 us
// forward (5.1 TB/s), 79 backward (5.2) and 6.4 for the 2048 parts of dw and db; 8191 x 8192
// bf16 97 (5.5), 116 (4.6) and 10.6; 1024 x 32768 52 and 99 (the backward reads h and dy
// for the rows' sums, for dx and for the columns' sums), 512 x 65536 88 and 119.
#include "nsa_launch.h"
#include "nsa_rows.h"

namespace nsa {

constexpr int kLnRegMax = 32768;         // widest row held in registers (forward)
constexpr int kLnBwdMax = 16384;         // ... and with its gradient and its parts of dw and db (backward)
constexpr int kLnMax = 1 << 24;          // widest row
constexpr int64_t kLnSlice = 1 << 21;    // rows of one launch

struct LnArgs {
  const void *x, *res, *w, *b;
  void *h, *y;
  float* stat;      // [rows][2]: mean, rstd; or null
  int64_t rows;
  int D;
  float eps, inv_d;
  double inv_d64;
  bool w_bf16, y_bf16;
};

// A run of 8 elements as it lies in memory, `n` of them in the row: of rows in which every
// thread's runs are whole, of others, and of rows of less than 8 elements.  The run at a
// row's end is asked for as the row's last 8 elements, like any other, and shifted when it
// is used: an element at a time it would hold up all loads behind it (66974 x 501 bf16,
// backward: 186 us so, 75 now).
enum { kWhole, kEdge, kTiny };
template <int EDGE>
struct RunAt {
  uint32_t off;   // what is loaded, from the row's first element on
  int n;
  __device__ __forceinline__ RunAt(int D, int c) : off((uint32_t)(EDGE == kEdge && D - c < 8 ? D - 8 : c)), n(D - c) {}
};
template <typename T>
struct RawRun {
  typedef T vec __attribute__((ext_vector_type(8), aligned(sizeof(T))));
  vec v;
  template <int EDGE>
  __device__ __forceinline__ void load(const T* row, const RunAt<EDGE>& at) {
    if constexpr (EDGE != kTiny) {
      v = *reinterpret_cast<const vec*>(row + at.off);
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j) v[j] = j < at.n ? row[at.off + j] : (T)0.0f;
    }
  }
  template <int EDGE>
  __device__ __forceinline__ void get(float (&f)[8], const RunAt<EDGE>& at) const {
#pragma unroll
    for (int j = 0; j < 8; ++j) f[j] = (float)v[j];
    if constexpr (EDGE == kEdge) {
      if (at.n > 0 && at.n < 8) {
        const int by = 8 - at.n;
#pragma unroll
        for (int k = 4; k >= 1; k >>= 1)
#pragma unroll
          for (int j = 0; j < 8; ++j) f[j] = by & k ? (j + k < 8 ? f[j + k] : 0.0f) : f[j];
      }
#pragma unroll
      for (int j = 0; j < 8; ++j) f[j] = at.n > 0 ? f[j] : 0.0f;
    }
  }
};
// Weights, of either type.
template <int EDGE>
__device__ __forceinline__ void ln_weights(const void* w, bool is_bf16, const RunAt<EDGE>& at, float (&f)[8]) {
  if (is_bf16) {
    RawRun<bf16> r;
    r.load(static_cast<const bf16*>(w), at);
    r.get(f, at);
  } else {
    RawRun<float> r;
    r.load(static_cast<const float*>(w), at);
    r.get(f, at);
  }
}

// Sums of K values over a row's threads: TPR of them, or past a wave the workgroup's
// (whole waves, TPR at most).  buf: K * TPR / 64 values.
template <int TPR, typename T, int K>
__device__ __forceinline__ void row_sums(T (&v)[K], T* buf) {
  static_assert(TPR <= 16 * kWave, "sixteen waves");
#pragma unroll
  for (int k = 0; k < K; ++k) v[k] = wave_sum<(TPR < kWave ? TPR : kWave)>(v[k]);
  if (TPR <= kWave) return;
  const int tid = threadIdx.x;
  if ((tid & (kWave - 1)) == 0) {
#pragma unroll
    for (int k = 0; k < K; ++k) buf[K * (tid / kWave) + k] = v[k];
  }
  __syncthreads();
  // (every lane of 16 takes one wave's)
  const int i = tid & 15;
  const bool there = i < (int)(blockDim.x / kWave);
#pragma unroll
  for (int k = 0; k < K; ++k) v[k] = wave_sum<16>(there ? buf[K * i + k] : (T)0);
}

// h of one run: x + r rounded to r's type (RES), or x itself
template <typename XT, typename RT, bool RES, int EDGE>
__device__ __forceinline__ void ln_sum8(const LnArgs& a, int64_t base, const RunAt<EDGE>& at, float (&h)[8]) {
  RawRun<XT> x;
  RawRun<RT> res;
  x.load(static_cast<const XT*>(a.x) + base, at);
  if (RES) res.load(static_cast<const RT*>(a.res) + base, at);
  x.get(h, at);
  if (RES) {
    float r[8];
    res.get(r, at);
#pragma unroll
    for (int j = 0; j < 8; ++j) h[j] = (float)(RT)(h[j] + r[j]);
  }
}

// TPR threads a row (past 64: the workgroup's, TPR at most), NV runs of 8 a thread (NV = 0:
// any length, h formed again for every pass).
template <typename XT, typename RT, bool RES, int TPR, int NV, int EDGE>
__global__ __launch_bounds__(TPR <= 64 ? 256 : TPR) void k_ln_fwd(const LnArgs a) {
  constexpr int W = TPR > kWave ? TPR / kWave : 1;
  __shared__ double red64[W];
  __shared__ float red[W];
  const int nth = TPR <= 64 ? TPR : (int)blockDim.x, t = TPR <= 64 ? threadIdx.x & (TPR - 1) : threadIdx.x;
  const int64_t row = TPR <= 64 ? (int64_t)blockIdx.x * (256 / TPR) + threadIdx.x / TPR : (int64_t)blockIdx.x;
  if (TPR <= 64 && row >= a.rows) return;   // (all of a row's lanes; no barrier follows for these)
  const int D = a.D;
  const int64_t base = row * D;
  const int nrun = NV > 0 ? NV : (D + 8 * nth - 1) / (8 * nth);
  float h[NV > 0 ? NV : 1][8];
  double s[1] = {0.0};
#pragma unroll
  for (int i = 0; i < nrun; ++i) {
    float(&hi)[8] = h[NV > 0 ? i : 0];
    const int c = 8 * (i * nth + t), n = D - c;
    ln_sum8<XT, RT, RES>(a, base, RunAt<EDGE>(D, c), hi);
    double q[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) q[j] = (double)hi[j];
    s[0] += ((q[0] + q[1]) + (q[2] + q[3])) + ((q[4] + q[5]) + (q[6] + q[7]));
    if (RES && n > 0) store_run8(static_cast<RT*>(a.h) + base + c, n, hi);
  }
  row_sums<TPR>(s, red64);
  const float mu = (float)(s[0] * a.inv_d64);
  float ss[1] = {0.0f};
#pragma unroll
  for (int i = 0; i < nrun; ++i) {
    float(&hi)[8] = h[NV > 0 ? i : 0];
    const int c = 8 * (i * nth + t), n = D - c;
    if (NV == 0) ln_sum8<XT, RT, RES>(a, base, RunAt<EDGE>(D, c), hi);
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      hi[j] -= mu;
      ss[0] += j < n ? hi[j] * hi[j] : 0.0f;
    }
  }
  row_sums<TPR>(ss, red);
  const float rstd = 1.0f / sqrtf(ss[0] * a.inv_d + a.eps);
  if (a.stat != nullptr && t == 0) {
    a.stat[2 * row] = mu;
    a.stat[2 * row + 1] = rstd;
  }
#pragma unroll
  for (int i = 0; i < nrun; ++i) {
    float(&hi)[8] = h[NV > 0 ? i : 0];
    const int c = 8 * (i * nth + t), n = D - c;
    if (NV == 0) {
      ln_sum8<XT, RT, RES>(a, base, RunAt<EDGE>(D, c), hi);
#pragma unroll
      for (int j = 0; j < 8; ++j) hi[j] -= mu;
    }
    float wv[8], bv[8] = {0, 0, 0, 0, 0, 0, 0, 0};
    ln_weights(a.w, a.w_bf16, RunAt<EDGE>(D, c), wv);
    if (a.b != nullptr) ln_weights(a.b, a.w_bf16, RunAt<EDGE>(D, c), bv);
#pragma unroll
    for (int j = 0; j < 8; ++j) hi[j] = (hi[j] * rstd) * wv[j] + bv[j];
    if (n > 0) {
      if (a.y_bf16)
        store_run8(static_cast<bf16*>(a.y) + base + c, n, hi);
      else
        store_run8(static_cast<float*>(a.y) + base + c, n, hi);
    }
  }
}

struct LnBwdArgs {
  const void *dy, *dh, *h, *w;
  const float* stat;
  void *dx, *dres;
  float* part;            // [2][gridDim.x][D] (dw, db), or null
  int64_t rows;
  int D;
  float inv_d;
  bool w_bf16, dx_bf16;
};

// YT: dy; RT: h, dh and dres.  dres is null where dx serves both (one type).
template <typename YT, typename RT, int TPR, int NV, int EDGE>
__global__ __launch_bounds__(TPR <= 64 ? 256 : TPR) void k_ln_bwd(const LnBwdArgs a) {
  constexpr int W = TPR > kWave ? TPR / kWave : 1;
  constexpr int RPG = TPR <= 64 ? 256 / TPR : 1;   // rows at a time
  __shared__ float red[2][2 * W];
  __shared__ float sums[RPG > 1 ? 8 * TPR * NV : 1];
  const int nth = TPR <= 64 ? TPR : (int)blockDim.x, t = TPR <= 64 ? threadIdx.x & (TPR - 1) : threadIdx.x;
  const int sub = TPR <= 64 ? threadIdx.x / TPR : 0;
  const int D = a.D;
  auto run_at = [&](int i) { return RunAt<EDGE>(D, 8 * (i * nth + t)); };
  // where the registers hold them: the weights for all rows, and dh asked for with the rest of a row
  constexpr bool kHold = NV * TPR <= 1024;
  float w[kHold ? NV : 1][8], dw[NV][8], db[NV][8];
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    if (kHold) ln_weights(a.w, a.w_bf16, run_at(i), w[kHold ? i : 0]);
#pragma unroll
    for (int j = 0; j < 8; ++j) dw[i][j] = db[i][j] = 0.0f;
  }
  int turn = 0;
  const int64_t step = (int64_t)gridDim.x * RPG;
  // a row of several waves is asked for before the sums of the row ahead of it, whose barrier
  // would leave the memory idle; wider rows (two runs a thread) have no registers for that
  constexpr bool kNext = kHold && TPR > kWave;
  struct Run {
    RawRun<RT> h, d;
    RawRun<YT> g;
  } ahead[kHold ? NV : 1];
  float mu_next = 0.0f, rstd_next = 0.0f;
  auto ask = [&](int64_t row) {
    const int64_t base = row * D;
#pragma unroll
    for (int i = 0; i < (kHold ? NV : 0); ++i) {
      const RunAt<EDGE> at = run_at(i);
      ahead[i].h.load(static_cast<const RT*>(a.h) + base, at);
      ahead[i].g.load(static_cast<const YT*>(a.dy) + base, at);
      if (a.dh != nullptr) ahead[i].d.load(static_cast<const RT*>(a.dh) + base, at);
    }
    mu_next = a.stat[2 * row];
    rstd_next = a.stat[2 * row + 1];
  };
  int64_t row = (int64_t)blockIdx.x * RPG + sub;
  if (kNext && row < a.rows) ask(row);
  for (; row < a.rows; row += step) {
    const int64_t base = row * D;
    if (!kNext) ask(row);
    const float mu = mu_next, rstd = rstd_next;
    float n_[NV][8], g[NV][8], d[kHold ? NV : 1][8];
    float sum[2] = {0.0f, 0.0f};
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const RunAt<EDGE> at = run_at(i);
      if constexpr (kHold) {
        ahead[i].h.get(n_[i], at);
        ahead[i].g.get(g[i], at);
        if (a.dh != nullptr) {
          ahead[i].d.get(d[i], at);
        } else {
#pragma unroll
          for (int j = 0; j < 8; ++j) d[i][j] = 0.0f;
        }
      } else {
        Run& r = ahead[0];
        r.h.load(static_cast<const RT*>(a.h) + base, at);
        r.g.load(static_cast<const YT*>(a.dy) + base, at);
        r.h.get(n_[i], at);
        r.g.get(g[i], at);
      }
    }
    if (kNext && row + step < a.rows) ask(row + step);
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      float(&wi)[8] = w[kHold ? i : 0];
      if (!kHold) ln_weights(a.w, a.w_bf16, run_at(i), wi);
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        n_[i][j] = (n_[i][j] - mu) * rstd;
        db[i][j] += g[i][j];
        dw[i][j] += g[i][j] * n_[i][j];
        g[i][j] *= wi[j];
        sum[0] += g[i][j];
        sum[1] += g[i][j] * n_[i][j];
      }
    }
    // two buffers in turn: the next row's sums are not written over those still being read
    row_sums<TPR>(sum, red[turn & 1]);
    const float s1 = sum[0] * a.inv_d, s2 = sum[1] * a.inv_d;
    ++turn;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int c = 8 * (i * nth + t), n = D - c;
      float(&di)[8] = d[kHold ? i : 0];
      if (!kHold) {
#pragma unroll
        for (int j = 0; j < 8; ++j) di[j] = 0.0f;
        if (a.dh != nullptr) {
          ahead[0].d.load(static_cast<const RT*>(a.dh) + base, run_at(i));
          ahead[0].d.get(di, run_at(i));
        }
      }
#pragma unroll
      for (int j = 0; j < 8; ++j) di[j] += rstd * (g[i][j] - s1 - n_[i][j] * s2);
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
  const int64_t next = (int64_t)gridDim.x * D;   // db's parts behind dw's
  if constexpr (RPG == 1) {
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int c = 8 * (i * nth + t);
      if (c < D) {
        store_run8(out + c, D - c, dw[i]);
        store_run8(out + next + c, D - c, db[i]);
      }
    }
  } else {
    static_assert(NV == 1, "a row of at most a wave is one run a lane");
    // the rows of a wave by halves, then the waves' parts in wave order
    const int wv = threadIdx.x / kWave;
    auto join = [&](float(&v)[8], float* dst) {
#pragma unroll
      for (int x = TPR; x < kWave; x <<= 1)
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] += __shfl_xor(v[j], x, kWave);
      for (int s = 0; s < 4; ++s) {
        if (wv == s && (threadIdx.x & (kWave - 1)) < TPR) {
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            const int c = 8 * t + j;
            if (c < D) sums[c] = s == 0 ? v[j] : sums[c] + v[j];
          }
        }
        __syncthreads();
      }
      for (int c = threadIdx.x; c < D; c += 256) dst[c] = sums[c];
    };
    join(dw[0], out);
    __syncthreads();
    join(db[0], out + next);
  }
}

// Rows past kLnBwdMax: one workgroup a row, read twice.
template <typename YT, typename RT>
__global__ __launch_bounds__(1024) void k_ln_bwd_long(const LnBwdArgs a) {
  __shared__ float red[2][32];   // (rows past kLnBwdMax only: wide)
  const int D = a.D;
  int turn = 0;
  for (int64_t row = blockIdx.x; row < a.rows; row += gridDim.x, ++turn) {
    const int64_t base = row * D;
    const float mu = a.stat[2 * row], rstd = a.stat[2 * row + 1];
    float sum[2] = {0.0f, 0.0f};
    for (int c = 8 * threadIdx.x; c < D; c += 8 * 1024) {
      float h[8], g[8], w[8];
      load_run8(static_cast<const RT*>(a.h) + base + c, D - c, h);
      load_run8(static_cast<const YT*>(a.dy) + base + c, D - c, g);
      load_run8_of(a.w, a.w_bf16, c, D - c, w);
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const float v = g[j] * w[j];
        sum[0] += v;
        sum[1] += v * ((h[j] - mu) * rstd);
      }
    }
    row_sums<1024>(sum, red[turn & 1]);
    const float s1 = sum[0] * a.inv_d, s2 = sum[1] * a.inv_d;
    for (int c = 8 * threadIdx.x; c < D; c += 8 * 1024) {
      const int n = D - c;
      float h[8], g[8], w[8], d[8] = {0, 0, 0, 0, 0, 0, 0, 0};
      load_run8(static_cast<const RT*>(a.h) + base + c, n, h);
      load_run8(static_cast<const YT*>(a.dy) + base + c, n, g);
      load_run8_of(a.w, a.w_bf16, c, n, w);
      if (a.dh != nullptr) load_run8(static_cast<const RT*>(a.dh) + base + c, n, d);
#pragma unroll
      for (int j = 0; j < 8; ++j) d[j] += rstd * (g[j] * w[j] - s1 - (h[j] - mu) * rstd * s2);
      if (a.dx_bf16)
        store_run8(static_cast<bf16*>(a.dx) + base + c, n, d);
      else
        store_run8(static_cast<float*>(a.dx) + base + c, n, d);
      if (a.dres != nullptr) store_run8(static_cast<RT*>(a.dres) + base + c, n, d);
    }
  }
}

// Parts of dw and db for such rows: 2048 columns and every gridDim.y-th row a workgroup.
template <typename YT, typename RT>
__global__ __launch_bounds__(256) void k_ln_dw_wide(const LnBwdArgs a) {
  const int c = 8 * ((int)blockIdx.x * 256 + (int)threadIdx.x), n = a.D - c;
  if (n <= 0) return;
  float dw[8] = {0, 0, 0, 0, 0, 0, 0, 0}, db[8] = {0, 0, 0, 0, 0, 0, 0, 0};
#pragma unroll 2
  for (int64_t row = blockIdx.y; row < a.rows; row += gridDim.y) {
    float h[8], g[8];
    load_run8(static_cast<const RT*>(a.h) + row * a.D + c, n, h);
    load_run8(static_cast<const YT*>(a.dy) + row * a.D + c, n, g);
    const float mu = a.stat[2 * row], rstd = a.stat[2 * row + 1];
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      dw[j] += g[j] * ((h[j] - mu) * rstd);
      db[j] += g[j];
    }
  }
  store_run8(a.part + (int64_t)blockIdx.y * a.D + c, n, dw);
  store_run8(a.part + ((int64_t)gridDim.y + blockIdx.y) * a.D + c, n, db);
}

// out[c] = sum of part[p][c] (dw for blockIdx.y = 0, db for 1): 32 columns a workgroup (a
// part's cache lines, each in one L2: 512 parts of 8192 8.4 us in a loop, 13.8 with half lines), 32
// interleaved sums over the parts, added in order.
__global__ __launch_bounds__(1024) void k_ln_dw(const float* __restrict__ part, int nparts, int D, void* dw, void* db,
                                                bool w_bf16) {
  __shared__ float acc[32][33];
  const int x = threadIdx.x & 31, s = threadIdx.x >> 5;
  const int c = blockIdx.x * 32 + x;
  void* out = blockIdx.y == 0 ? dw : db;
  if (out == nullptr) return;
  part += (int64_t)blockIdx.y * nparts * D;
  float v = 0.0f;
  if (c < D) {
#pragma unroll 8
    for (int p = s; p < nparts; p += 32) v += part[(int64_t)p * D + c];
  }
  acc[s][x] = v;
  __syncthreads();
  if (s < 2) {   // 16 sums each by the halves of the first wave, then those two
    float t = 0.0f;
#pragma unroll
    for (int i = 0; i < 16; ++i) t += acc[16 * s + i][x];
    t += __shfl_xor(t, 32, kWave);
    if (s == 0 && c < D) {
      if (w_bf16)
        static_cast<bf16*>(out)[c] = (bf16)t;
      else
        static_cast<float*>(out)[c] = t;
    }
  }
}

// Threads a row (the most, from which the kernel's registers follow) and runs a thread:
// the fewest threads that hold the row with one run each; past 8192 elements two or
// four runs.  Past a wave as many waves are launched as the row needs (8184 x 4100
// bf16 in 9 waves: forward 46 us, backward 76; 75 and 110 in 16).
struct LnShape {
  int tpr, nv;
};
#define NSA_LN_SHAPES(X) X(8, 1) X(16, 1) X(32, 1) X(64, 1) X(128, 1) X(256, 1) X(512, 1) X(1024, 1) X(1024, 2)
static LnShape ln_shape(int D) {
  const int runs = (D + 7) / 8;
#define NSA_LN_FITS(TPR, NV) \
  if (runs <= TPR * NV) return {TPR, NV};
  NSA_LN_SHAPES(NSA_LN_FITS)
#undef NSA_LN_FITS
  return {1024, D <= kLnRegMax ? 4 : 0};
}

static int ln_threads(LnShape s, int D) {
  if (s.tpr <= 64) return 256;
  if (s.nv == 0) return s.tpr;
  return ((D + 7) / 8 + s.nv * kWave - 1) / (s.nv * kWave) * kWave;
}

// How a row's runs lie in its threads
template <int TPR, typename F>
static void ln_edge(LnShape s, int D, F f) {
  const int threads = TPR <= 64 ? TPR : ln_threads(s, D);
  if (D == threads * s.nv * 8) return f(std::integral_constant<int, kWhole>{});
  if constexpr (TPR == 8) {
    if (D < 8) return f(std::integral_constant<int, kTiny>{});
  }
  f(std::integral_constant<int, kEdge>{});
}

template <typename XT, typename RT, bool RES>
static int ln_fwd_launch(const LnArgs& a, hipStream_t s) {
  const LnShape sh = ln_shape(a.D);
  const int threads = ln_threads(sh, a.D);
#define NSA_LN_CASE(TPR, NV)                                                                                   \
  if (sh.tpr == TPR && sh.nv == NV) {                                                                          \
    const unsigned grid = (unsigned)(TPR <= 64 ? (a.rows + 256 / TPR - 1) / (256 / TPR) : a.rows);             \
    ln_edge<TPR>(sh, a.D, [&](auto e) {                                                                        \
      k_ln_fwd<XT, RT, RES, TPR, NV, decltype(e)::value><<<grid, threads, 0, s>>>(a);                          \
    });                                                                                                        \
    return nsa_launch_status();                                                                                \
  }
  NSA_LN_SHAPES(NSA_LN_CASE) NSA_LN_CASE(1024, 4) NSA_LN_CASE(1024, 0)
#undef NSA_LN_CASE
  return NSA_ERR_SHAPE;
}

template <typename XT, typename RT>
static int ln_fwd_as(const LnArgs& a, hipStream_t s) {
  if (a.res != nullptr) return ln_fwd_launch<XT, RT, true>(a, s);
  if constexpr (sizeof(XT) == sizeof(RT)) return ln_fwd_launch<XT, RT, false>(a, s);
  return NSA_ERR_DTYPE;
}

// Parts of dw and db: a workgroup of the backward each; past kLnBwdMax a row group of
// k_ln_dw_wide.  A part is written and read once more, 16 bytes an element against the 8 or 16
// of a row's in bf16 or float32: workgroups take 16 rows in turn (4 where rows are few), while
// they are eight waves a compute unit and one workgroup each, and no more than the chip holds
// (bf16, 2048 x 768 10 us, 16.5 with a row each; 4096 x 4096 26 and 36; 8192 x 2048 26 and 35).
static int64_t ln_bwd_groups(int64_t rows, int D, int cu) {
  if (D > kLnBwdMax) return rows < 128 ? rows : 128;
  const LnShape sh = ln_shape(D);
  const int rpg = sh.tpr <= 64 ? 256 / sh.tpr : 1, threads = ln_threads(sh, D);
  const int64_t turns = (rows + rpg - 1) / rpg;   // of one workgroup
  const int64_t most = (int64_t)cu * (threads <= 256 ? 8 : 2048 / threads), eight = (int64_t)cu * 512 / threads;
  int64_t groups = turns / 16 > eight ? turns / 16 : eight;
  groups = groups < turns / 4 ? groups : turns / 4;
  groups = groups > cu ? groups : cu;
  groups = groups < most ? groups : most;
  return groups < turns ? groups : turns;
}

template <typename YT, typename RT>
static int ln_bwd_launch(LnBwdArgs a, void* dw, void* db, hipStream_t s) {
  const int cu = device_cu_count(s);
  const LnShape sh = ln_shape(a.D);
  const int64_t grid = ln_bwd_groups(a.rows, a.D, cu);
  bool done = false;
  if (a.D > kLnBwdMax) {
    k_ln_bwd_long<YT, RT><<<(unsigned)(a.rows < 8192 ? a.rows : 8192), 1024, 0, s>>>(a);
    if (a.part != nullptr)
      k_ln_dw_wide<YT, RT><<<dim3((unsigned)((a.D + 2047) / 2048), (unsigned)grid), 256, 0, s>>>(a);
    done = true;
  }
  const int threads = ln_threads(sh, a.D);
#define NSA_LN_CASE(TPR, NV)                                                                       \
  if (!done && sh.tpr == TPR && sh.nv == NV) {                                                     \
    ln_edge<TPR>(sh, a.D, [&](auto e) {                                                            \
      k_ln_bwd<YT, RT, TPR, NV, decltype(e)::value><<<(unsigned)grid, threads, 0, s>>>(a);         \
    });                                                                                            \
    done = true;                                                                                   \
  }
  NSA_LN_SHAPES(NSA_LN_CASE)
#undef NSA_LN_CASE
  if (!done) return NSA_ERR_SHAPE;
  if (a.part != nullptr)
    k_ln_dw<<<dim3((unsigned)((a.D + 31) / 32), 2), 1024, 0, s>>>(a.part, (int)grid, a.D, dw, db, a.w_bf16);
  return nsa_launch_status();
}

static bool ln_type(int dtype) { return dtype == NSA_F32 || dtype == NSA_BF16; }

}  // namespace nsa

extern "C" int nsa_lnorm_fwd(const void* x, const void* res, const void* w, const void* b, void* h, void* y,
                             float* stat, int64_t rows, int D, float eps, int x_dtype, int h_dtype, int w_dtype,
                             int y_dtype, void* stream) {
  using namespace nsa;
  NSA_CHECK(rows >= 0 && rows <= 0x7fffffffLL && D >= 1 && D <= kLnMax, NSA_ERR_SHAPE);
  NSA_CHECK(ln_type(x_dtype) && ln_type(h_dtype) && ln_type(w_dtype) && ln_type(y_dtype), NSA_ERR_DTYPE);
  NSA_CHECK(res != nullptr || x_dtype == h_dtype, NSA_ERR_DTYPE);
  if (rows == 0) return NSA_OK;
  NSA_CHECK(x != nullptr && w != nullptr && y != nullptr, NSA_ERR_ARG);
  NSA_CHECK(res == nullptr || h != nullptr, NSA_ERR_ARG);
  const hipStream_t s = static_cast<hipStream_t>(stream);
  const size_t xs = x_dtype == NSA_BF16 ? 2 : 4, hs = h_dtype == NSA_BF16 ? 2 : 4, ys = y_dtype == NSA_BF16 ? 2 : 4;
  // 2^21 rows a launch: a grid holds less than 2^32 threads
  for (int64_t r0 = 0; r0 < rows; r0 += kLnSlice) {
    const int64_t n = rows - r0 < kLnSlice ? rows - r0 : kLnSlice, at = r0 * D;
    const LnArgs a{static_cast<const char*>(x) + at * xs,
                   res == nullptr ? nullptr : static_cast<const char*>(res) + at * hs,
                   w,
                   b,
                   h == nullptr ? nullptr : static_cast<char*>(h) + at * hs,
                   static_cast<char*>(y) + at * ys,
                   stat == nullptr ? nullptr : stat + 2 * r0,
                   n, D, eps, 1.0f / (float)D, 1.0 / (double)D, w_dtype == NSA_BF16, y_dtype == NSA_BF16};
    int rc;
    if (x_dtype == NSA_BF16)
      rc = h_dtype == NSA_BF16 ? ln_fwd_as<bf16, bf16>(a, s) : ln_fwd_as<bf16, float>(a, s);
    else
      rc = h_dtype == NSA_BF16 ? ln_fwd_as<float, bf16>(a, s) : ln_fwd_as<float, float>(a, s);
    if (rc != NSA_OK) return rc;
  }
  return NSA_OK;
}

extern "C" size_t nsa_lnorm_bwd_workspace(int64_t rows, int D, void* stream) {
  using namespace nsa;
  if (rows < 0 || rows > 0x7fffffffLL || D < 1 || D > kLnMax) return 0;
  if (rows == 0) return 16;
  return (size_t)ln_bwd_groups(rows, D, device_cu_count(static_cast<hipStream_t>(stream))) * D * 2 * sizeof(float);
}

extern "C" int nsa_lnorm_bwd(const void* dy, const void* dh, const void* h, const void* w, const float* stat, void* dx,
                             void* dres, void* dw, void* db, void* workspace, size_t workspace_bytes, int64_t rows,
                             int D, int x_dtype, int h_dtype, int w_dtype, int y_dtype, void* stream) {
  using namespace nsa;
  NSA_CHECK(rows >= 1 && rows <= 0x7fffffffLL && D >= 1 && D <= kLnMax, NSA_ERR_SHAPE);
  NSA_CHECK(ln_type(x_dtype) && ln_type(h_dtype) && ln_type(w_dtype) && ln_type(y_dtype), NSA_ERR_DTYPE);
  NSA_CHECK(dy != nullptr && h != nullptr && w != nullptr && stat != nullptr && dx != nullptr, NSA_ERR_ARG);
  const hipStream_t s = static_cast<hipStream_t>(stream);
  float* part = nullptr;
  if (dw != nullptr || db != nullptr) {
    NSA_CHECK(workspace != nullptr && workspace_bytes >= nsa_lnorm_bwd_workspace(rows, D, stream), NSA_ERR_WORKSPACE);
    part = static_cast<float*>(workspace);
  }
  const LnBwdArgs a{dy, dh, h, w, stat, dx, dres, part, rows, D, 1.0f / (float)D, w_dtype == NSA_BF16,
                    x_dtype == NSA_BF16};
  if (y_dtype == NSA_BF16)
    return h_dtype == NSA_BF16 ? ln_bwd_launch<bf16, bf16>(a, dw, db, s) : ln_bwd_launch<bf16, float>(a, dw, db, s);
  return h_dtype == NSA_BF16 ? ln_bwd_launch<float, bf16>(a, dw, db, s) : ln_bwd_launch<float, float>(a, dw, db, s);
}
