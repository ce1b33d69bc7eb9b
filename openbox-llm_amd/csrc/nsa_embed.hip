// Rows of a table by token, with a row of a second table by position:
//
//   out[i] = scale W[t_i] + P[p_i]     (float32, rounded once)
//   dW[v] = scale sum over {i: t_i = v} of dy[i],   dP[p] = sum over {i: p_i = p} of dy[i]
//
// A token (position) outside its table is none: it adds nothing and has no gradient.
//
// The gradient of a table is dense, has the same bits on every run and is bound by
// the bytes of dy and of the table.  It goes by sorted tokens:
//
//   1. (token, i) pairs are sorted by token with ties by ascending i: a radix sort
//      of up to 9 bits a pass, each pass two launches (counts of every block of
//      pairs; places from the counts, ranks within a wave by ballots), or one launch
//      of one workgroup for up to 4096 pairs.  Positions
//      0 .. T-1 of every sequence need no sort: the sorted list is a formula.
//   2. The sorted list is cut into pieces of equal length, whatever the tokens'
//      frequencies (in text one token can be a tenth of all): a workgroup adds the
//      rows of its piece one after another and writes a token's row where the run
//      of the token ends.  A run that is cut leaves its parts in float32.  Other
//      workgroups of the same launch clear the rows without a token, so that the
//      table is written once.
//   3. The parts of every cut run are added in the order of the pieces.
//
// The same lists give sums of weighted rows by token (nsa_token_sums), for the gradient of
// a head's weights: a token's sum then lies at its run's place in the sorted list.
//
// Measured: 8 x 4096 rows of 768 in float32 with their positions, table of 32000: 38 us
// forward (300 MB less what the caches hold of the table; a copy's rate is 5.4 TB/s); 49 for
// the tokens' sums (200 MB, 4.1 TB/s), 20 for their sort (four launches of one dependent
// chain each), 11 for the joins, 18 for the positions' sums. 8191 x 4096 bf16 rows: 22 us.
#include <utility>

#include "nsa_launch.h"
#include "nsa_rows.h"

namespace nsa {

constexpr int64_t kEmbedRows = 0x7ffffff0LL;    // most tokens, and most rows of a table
constexpr int kEmbedWide = 1 << 20;             // widest row

struct EmbedArgs {
  const int64_t *tokens, *pos;
  const void *w, *pw;
  void* out;
  int64_t first, n, T, V, P;   // rows first .. n - 1
  int D;
  float scale;
  bool w_bf16, pw_bf16, out_bf16;
};

// E elements at any element-aligned address, `n` of them in the row from here on; a
// float32 row goes by 4 a lane, so that neighbouring lanes' 16 bytes are neighbours.
template <int E>
__device__ __forceinline__ void load_some(const void* p, bool is_bf16, int64_t at, int n, float (&f)[E]) {
  typedef bf16 bf16xE __attribute__((ext_vector_type(E), aligned(2)));
  typedef float f32xE __attribute__((ext_vector_type(E), aligned(4)));
  if (n >= E) {
    if (is_bf16) {
      const bf16xE v = *reinterpret_cast<const bf16xE*>(static_cast<const bf16*>(p) + at);
#pragma unroll
      for (int j = 0; j < E; ++j) f[j] = (float)v[j];
    } else {
      const f32xE v = *reinterpret_cast<const f32xE*>(static_cast<const float*>(p) + at);
#pragma unroll
      for (int j = 0; j < E; ++j) f[j] = v[j];
    }
  } else {
#pragma unroll
    for (int j = 0; j < E; ++j)
      f[j] = j >= n ? 0.0f : is_bf16 ? (float)static_cast<const bf16*>(p)[at + j] : static_cast<const float*>(p)[at + j];
  }
}
// (PAST: the caches keep nothing of it)
template <int E, bool PAST = false>
__device__ __forceinline__ void store_some(void* p, bool is_bf16, int64_t at, int n, const float (&f)[E]) {
  typedef bf16 bf16xE __attribute__((ext_vector_type(E), aligned(2)));
  typedef float f32xE __attribute__((ext_vector_type(E), aligned(4)));
  if (n >= E) {
    if (is_bf16) {
      bf16xE v;
#pragma unroll
      for (int j = 0; j < E; ++j) v[j] = (bf16)f[j];
      if (PAST)
        __builtin_nontemporal_store(v, reinterpret_cast<bf16xE*>(static_cast<bf16*>(p) + at));
      else
        *reinterpret_cast<bf16xE*>(static_cast<bf16*>(p) + at) = v;
    } else {
      f32xE v;
#pragma unroll
      for (int j = 0; j < E; ++j) v[j] = f[j];
      if (PAST)
        __builtin_nontemporal_store(v, reinterpret_cast<f32xE*>(static_cast<float*>(p) + at));
      else
        *reinterpret_cast<f32xE*>(static_cast<float*>(p) + at) = v;
    }
  } else {
#pragma unroll
    for (int j = 0; j < E; ++j)
      if (j < n) {
        if (is_bf16)
          static_cast<bf16*>(p)[at + j] = (bf16)f[j];
        else
          static_cast<float*>(p)[at + j] = f[j];
      }
  }
}

// Where the run of E columns from c < D on is taken: at a row's end the last E columns,
// with the same values as the run before it has for them (an element at a time the odd
// ones hold up the others: 65536 bf16 rows of 765 take 26 us, 38 so, the gradient 65 and 105).
template <int E>
__device__ __forceinline__ int run_start(int c, int D) {
  return D >= E && c > D - E ? D - E : c;
}

// TPR threads a row, 256 / TPR rows a workgroup; a thread has 16 elements of each table in flight.
template <int E, int TPR, bool PAST>
__global__ __launch_bounds__(256) void k_embed_fwd(const EmbedArgs a) {
  const int t = threadIdx.x & (TPR - 1);
  const int64_t i = a.first + (int64_t)blockIdx.x * (256 / TPR) + threadIdx.x / TPR;
  if (i >= a.n) return;
  const int64_t tok = a.tokens[i];
  const bool real = tok >= 0 && tok < a.V;
  // (fewer than 2^31 rows, and T too: a 32-bit remainder)
  const int64_t p = a.pw == nullptr ? 0 : a.pos != nullptr ? a.pos[i] : (int64_t)((uint32_t)i % (uint32_t)a.T);
  const bool has_pos = a.pw != nullptr && p >= 0 && p < a.P;
  const int D = a.D;
  constexpr int U = E == 4 ? 4 : 2;
  for (int c0 = E * t; c0 < D; c0 += U * E * TPR) {
    float v[U][E], q[U][E];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int cu = c0 + u * E * TPR, c = run_start<E>(cu, D);
#pragma unroll
      for (int j = 0; j < E; ++j) v[u][j] = q[u][j] = 0.0f;
      if (real && cu < D) load_some<E>(a.w, a.w_bf16, tok * D + c, D - c, v[u]);
      if (has_pos && cu < D) load_some<E>(a.pw, a.pw_bf16, p * D + c, D - c, q[u]);
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int cu = c0 + u * E * TPR, c = run_start<E>(cu, D);
#pragma unroll
      for (int j = 0; j < E; ++j) v[u][j] = real ? fmaf(v[u][j], a.scale, q[u][j]) : q[u][j];
      if (cu < D) store_some<E, PAST>(a.out, a.out_bf16, i * D + c, D - c, v[u]);
    }
  }
}

// ---------------------------------------------------------------------------
// sort of (key, i) by key, ties by i
// ---------------------------------------------------------------------------
constexpr int kSortThreads = 256;
constexpr int kSortWaves = kSortThreads / kWave;
constexpr int kSortBits = 9;
constexpr int kSortBins = 1 << kSortBits;
constexpr int kSortAhead = 4;   // pairs a thread asks for at a time; `per` is a multiple of it

struct SortPass {
  const int64_t* tokens;              // first pass: keys from here, i in order; else null
  const uint32_t *key_in, *val_in;
  uint32_t *key_out, *val_out;
  uint32_t* count;                    // [blocks][bins]
  int64_t n, V;
  int per, shift, bits;               // pairs a thread; the pass's digit
};

// The key of pair i: the token, or V (behind all tokens) for none.
__device__ __forceinline__ uint32_t sort_key(const SortPass& a, int64_t i) {
  if (a.tokens == nullptr) return a.key_in[i];
  const int64_t t = a.tokens[i];
  return (uint32_t)(t >= 0 && t < a.V ? t : a.V);
}

__global__ __launch_bounds__(kSortThreads) void k_sort_count(const SortPass a) {
  __shared__ uint32_t bins[kSortBins];
  const int nb = 1 << a.bits;
  for (int b = threadIdx.x; b < nb; b += kSortThreads) bins[b] = 0;
  __syncthreads();
  const int64_t first = (int64_t)blockIdx.x * kSortThreads * a.per;
  for (int r0 = 0; r0 < a.per; r0 += kSortAhead) {
    uint32_t key[kSortAhead];
#pragma unroll
    for (int u = 0; u < kSortAhead; ++u) {
      const int64_t i = first + (int64_t)(r0 + u) * kSortThreads + threadIdx.x;
      key[u] = i < a.n ? sort_key(a, i) : 0u;
    }
#pragma unroll
    for (int u = 0; u < kSortAhead; ++u) {
      const int64_t i = first + (int64_t)(r0 + u) * kSortThreads + threadIdx.x;
      if (i < a.n) atomicAdd(&bins[(key[u] >> a.shift) & (nb - 1)], 1u);
    }
  }
  __syncthreads();
  for (int b = threadIdx.x; b < nb; b += kSortThreads) a.count[(int64_t)blockIdx.x * nb + b] = bins[b];
}

// A wave owns per * 64 consecutive pairs of the block and takes them 64 at a time.
__global__ __launch_bounds__(kSortThreads) void k_sort_move(const SortPass a) {
  __shared__ uint32_t seen[kSortWaves][kSortBins];   // pairs of a digit that a wave has met
  __shared__ uint32_t base[kSortBins];
  __shared__ uint32_t wsum[kSortWaves];
  const int nb = 1 << a.bits, tid = threadIdx.x, w = tid / kWave, lane = tid & (kWave - 1);
  const int64_t first = (int64_t)blockIdx.x * kSortThreads * a.per + (int64_t)w * kWave * a.per;
  auto at_of = [&](int r) { return first + (int64_t)r * kWave + lane; };
  uint32_t key[kSortAhead], val[kSortAhead];
  auto load = [&](int r0) {
#pragma unroll
    for (int u = 0; u < kSortAhead; ++u) {
      const int64_t i = at_of(r0 + u);
      key[u] = i < a.n ? sort_key(a, i) : 0u;
      val[u] = a.tokens != nullptr || i >= a.n ? (uint32_t)i : a.val_in[i];
    }
  };
  load(0);
  // places of the block's digits: all smaller digits, then this digit's earlier blocks
  constexpr int kPer = kSortBins / kSortThreads;
  uint32_t total[kPer], before[kPer], mine = 0;
  static_assert(kPer == 2, "two bins a thread");
  total[0] = total[1] = before[0] = before[1] = 0;
  if (2 * tid < nb) {
#pragma unroll 16
    for (int g = 0; g < (int)gridDim.x; ++g) {
      const uint2 c = *reinterpret_cast<const uint2*>(a.count + (int64_t)g * nb + 2 * tid);
      const bool earlier = g < (int)blockIdx.x;
      total[0] += c.x;
      total[1] += c.y;
      before[0] += earlier ? c.x : 0u;
      before[1] += earlier ? c.y : 0u;
    }
  }
  mine = total[0] + total[1];
  uint32_t incl = mine;
#pragma unroll
  for (int d = 1; d < kWave; d <<= 1) {
    const uint32_t o = __shfl_up(incl, d, kWave);
    if (lane >= d) incl += o;
  }
  if (lane == kWave - 1) wsum[w] = incl;
  for (int b = tid; b < kSortWaves * kSortBins; b += kSortThreads) (&seen[0][0])[b] = 0;
  __syncthreads();
  uint32_t at = incl - mine;
  for (int k = 0; k < w; ++k) at += wsum[k];
#pragma unroll
  for (int k = 0; k < kPer; ++k) {
    base[tid * kPer + k] = at + before[k];
    at += total[k];
  }
  // 1st walk: how many pairs of each digit every wave has
  for (int r0 = 0; r0 < a.per; r0 += kSortAhead) {
    if (r0 > 0) load(r0);
#pragma unroll
    for (int u = 0; u < kSortAhead; ++u)
      if (at_of(r0 + u) < a.n) atomicAdd(&seen[w][(key[u] >> a.shift) & (nb - 1)], 1u);
  }
  __syncthreads();
  // the waves' starts of each digit
  for (int b = tid; b < nb; b += kSortThreads) {
    uint32_t s = base[b];
#pragma unroll
    for (int k = 0; k < kSortWaves; ++k) {
      const uint32_t c = seen[k][b];
      seen[k][b] = s;
      s += c;
    }
  }
  __syncthreads();
  // 2nd walk: a pair's place is its wave's next of the digit, plus its rank among the 64
  for (int r0 = 0; r0 < a.per; r0 += kSortAhead) {
    if (a.per > kSortAhead) load(r0);
#pragma unroll
    for (int u = 0; u < kSortAhead; ++u) {
      const bool ok = at_of(r0 + u) < a.n;
      const uint32_t dig = (key[u] >> a.shift) & (nb - 1);
      uint64_t same = __ballot(ok);
      for (int b = 0; b < a.bits; ++b) {
        const uint64_t m = __ballot((dig >> b) & 1u);
        same &= (dig >> b) & 1u ? m : ~m;
      }
      if (ok) {
        const uint32_t to = seen[w][dig] + (uint32_t)__popcll(same & ((1ull << lane) - 1ull));
        a.key_out[to] = key[u];
        a.val_out[to] = val[u];
      }
      // (LDS accesses of a wave keep their order: all have read before one adds)
      __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
      if (ok && (same >> lane) == 1ull) seen[w][dig] += (uint32_t)__popcll(same);
      __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    }
  }
}

// All passes of up to kSmallSort pairs in one workgroup of 16 waves, the pairs in LDS.
constexpr int kSmallSort = 4096;
__global__ __launch_bounds__(1024) void k_sort_small(const int64_t* tokens, uint32_t* key_out, uint32_t* val_out, int n,
                                                     int64_t V, int passes, int bits) {
  constexpr int W = 16;
  __shared__ uint32_t key[2][kSmallSort], val[2][kSmallSort], seen[W][kSortBins], wsum[8];
  const int tid = threadIdx.x, w = tid / kWave, lane = tid & (kWave - 1);
  const int per = (n + 1023) / 1024, first = w * kWave * per;   // a wave owns `per` * 64 pairs in a row
  for (int i = tid; i < n; i += 1024) {
    const int64_t t = tokens[i];
    key[0][i] = (uint32_t)(t >= 0 && t < V ? t : V);
    val[0][i] = (uint32_t)i;
  }
  int from = 0, shift = 0;
  for (int q = 0; q < passes; ++q, from ^= 1) {
    const int b = (bits - shift + passes - q - 1) / (passes - q), nb = 1 << b;
    for (int i = tid; i < W * kSortBins; i += 1024) (&seen[0][0])[i] = 0;
    __syncthreads();
    for (int r = 0; r < per; ++r) {
      const int i = first + r * kWave + lane;
      if (i < n) atomicAdd(&seen[w][(key[from][i] >> shift) & (nb - 1)], 1u);
    }
    __syncthreads();
    // starts: all smaller digits, then the earlier waves
    uint32_t total = 0, incl = 0;
    if (tid < kSortBins) {
#pragma unroll
      for (int k = 0; k < W; ++k) total += seen[k][tid];
      incl = total;
#pragma unroll
      for (int d = 1; d < kWave; d <<= 1) {
        const uint32_t o = __shfl_up(incl, d, kWave);
        if (lane >= d) incl += o;
      }
      if (lane == kWave - 1) wsum[w] = incl;
    }
    __syncthreads();
    if (tid < kSortBins) {
      uint32_t at = incl - total;
      for (int k = 0; k < w; ++k) at += wsum[k];
#pragma unroll
      for (int k = 0; k < W; ++k) {
        const uint32_t c = seen[k][tid];
        seen[k][tid] = at;
        at += c;
      }
    }
    __syncthreads();
    for (int r = 0; r < per; ++r) {
      const int i = first + r * kWave + lane;
      const bool ok = i < n;
      const uint32_t k = ok ? key[from][i] : 0u, dig = (k >> shift) & (nb - 1);
      uint64_t same = __ballot(ok);
      for (int x = 0; x < b; ++x) {
        const uint64_t m = __ballot((dig >> x) & 1u);
        same &= (dig >> x) & 1u ? m : ~m;
      }
      if (ok) {
        const uint32_t to = seen[w][dig] + (uint32_t)__popcll(same & ((1ull << lane) - 1ull));
        key[from ^ 1][to] = k;
        val[from ^ 1][to] = val[from][i];
      }
      __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");   // (as in k_sort_move)
      if (ok && (same >> lane) == 1ull) seen[w][dig] += (uint32_t)__popcll(same);
      __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    }
    __syncthreads();
    shift += b;
  }
  for (int i = tid; i < n; i += 1024) {
    key_out[i] = key[from][i];
    val_out[i] = val[from][i];
  }
}

// ---------------------------------------------------------------------------
// sums over the runs of the sorted list
// ---------------------------------------------------------------------------
constexpr int kRunRows = 32;   // pairs of the sorted list in LDS
constexpr int kAhead = 8;      // rows asked for at a time

struct EmbedGrad {
  const uint32_t *key, *val;   // the sorted list; null: positions of B sequences of T
  const void* dy;
  void* dw;
  float* part;                 // [pieces][2][D]: the parts of a piece's first run and of its last
  int64_t n, T, V;
  uint32_t B;
  int D, len, pieces;          // len: pairs a piece
  float scale;
  bool dy_bf16, w_bf16;
  const float* weight;         // [n], sums by token: of every row; dw then has a row a pair, a run's at its first pair
  int* first;                  // [V], sums by token: a token's first pair, of those that have one,
  uint64_t* there;             // ... whose bits these are
  // (fewer than 2^31 pairs: 32-bit divisions)
  __device__ __forceinline__ uint32_t key_at(int64_t s) const { return key != nullptr ? key[s] : (uint32_t)s / B; }
  __device__ __forceinline__ uint32_t row_at(int64_t s) const {
    return key != nullptr ? val[s] : (uint32_t)s % B * (uint32_t)T + (uint32_t)s / B;
  }
};

template <int E>
__device__ __forceinline__ void embed_store(const EmbedGrad& a, int64_t at, int n, const float (&v)[E]) {
  float o[E];
#pragma unroll
  for (int j = 0; j < E; ++j) o[j] = v[j] * a.scale;
  store_some<E>(a.dw, a.w_bf16, at, n, o);
}

// Clear the rows r0 .. r0 + 63 that have no token, columns c ..  SUMS: note these tokens' first pairs.
template <int E, bool SUMS>
__device__ __forceinline__ void embed_clear(const EmbedGrad& a, int64_t r0, int c) {
  const int n = a.D - c;
  const int64_t v = r0 + (threadIdx.x & 63);
  bool empty = v < a.V;
  if (empty) {   // the first pair whose key is at least v
    int64_t lo = 0, hi = a.n;
    while (lo < hi) {
      const int64_t mid = (lo + hi) >> 1;
      if (a.key_at(mid) < (uint32_t)v)
        lo = mid + 1;
      else
        hi = mid;
    }
    empty = lo >= a.n || a.key_at(lo) != (uint32_t)v;
    if (SUMS && !empty && threadIdx.x < 64 && blockIdx.y == 0) a.first[v] = (int)lo;
  }
  if (SUMS) {
    const uint64_t there = __ballot(v < a.V && !empty);
    if (threadIdx.x == 0 && blockIdx.y == 0) a.there[r0 / 64] = there;
    return;
  }
  uint64_t rows = __ballot(empty);   // (every wave of the workgroup: the same)
  if (n <= 0) return;
  float zero[E];
#pragma unroll
  for (int j = 0; j < E; ++j) zero[j] = 0.0f;
  while (rows != 0) {
    const int64_t at = (r0 + __builtin_ctzll(rows)) * a.D + c;
    rows &= rows - 1;
    store_some<E>(a.dw, a.w_bf16, at, n, zero);
  }
}

// Workgroups below a.pieces add the rows of a piece; the others clear the rows
// without a token, 64 rows of the table at a time.  A thread owns E columns.
template <int E, bool SUMS>
__global__ __launch_bounds__(256) void k_embed_runs(const EmbedGrad a) {
  __shared__ uint32_t keys[kRunRows + 1], rows[kRunRows];
  __shared__ float weights[SUMS ? kRunRows : 1];
  const int tid = threadIdx.x, D = a.D;
  const int ct = ((int)blockIdx.y * (int)blockDim.x + tid) * E, c = ct < D ? run_start<E>(ct, D) : D, n = D - c;
  if ((int)blockIdx.x >= a.pieces) {
    for (int64_t r0 = ((int64_t)blockIdx.x - a.pieces) * 64; r0 < a.V; r0 += ((int64_t)gridDim.x - a.pieces) * 64)
      embed_clear<E, SUMS>(a, r0, c);
    return;
  }
  const int64_t s0 = (int64_t)blockIdx.x * a.len, s1 = s0 + a.len < a.n ? s0 + a.len : a.n;
  const uint32_t none = (uint32_t)a.V, end = none + 1;
  const uint32_t k_prev = s0 > 0 ? a.key_at(s0 - 1) : end, k_next = s1 < a.n ? a.key_at(s1) : end;
  float* part = a.part + (int64_t)blockIdx.x * 2 * D;
  float acc[E];
#pragma unroll
  for (int j = 0; j < E; ++j) acc[j] = 0.0f;
  bool head = a.key_at(s0) == k_prev;   // the run began in an earlier piece
  int64_t start = s0;                   // ... else here
  for (int64_t s = s0; s < s1; s += kRunRows) {
    const int m = s1 - s < kRunRows ? (int)(s1 - s) : kRunRows;
    __syncthreads();
    if (tid <= m) keys[tid] = tid < m || s + m < s1 ? a.key_at(s + tid) : end;   // (the key behind each row; `end` behind the piece)
    if (tid < m) {
      rows[tid] = a.row_at(s + tid);
      if (SUMS) weights[tid] = a.weight[rows[tid]];
    }
    __syncthreads();
    if (n <= 0) continue;
    for (int u0 = 0; u0 < m; u0 += kAhead) {
      float v[kAhead][E];
#pragma unroll
      for (int u = 0; u < kAhead; ++u)
        if (u0 + u < m) load_some<E>(a.dy, a.dy_bf16, (int64_t)rows[u0 + u] * D + c, n, v[u]);
#pragma unroll
      for (int u = 0; u < kAhead; ++u) {
        if (u0 + u >= m) continue;
        const uint32_t k = keys[u0 + u], kn = keys[u0 + u + 1];
        if (k == none) continue;
#pragma unroll
        for (int j = 0; j < E; ++j) acc[j] = SUMS ? fmaf(weights[u0 + u], v[u][j], acc[j]) : acc[j] + v[u][j];
        if (kn == k) continue;
        if (head)
          store_some<E>(part, false, c, n, acc);
        else if (kn == end && k == k_next)   // the run goes on in the next piece
          store_some<E>(part, false, D + c, n, acc);
        else
          embed_store<E>(a, (SUMS ? start : (int64_t)k) * D + c, n, acc);
        head = false;
        start = s + u0 + u + 1;
#pragma unroll
        for (int j = 0; j < E; ++j) acc[j] = 0.0f;
      }
    }
  }
}

// The cut runs: a workgroup for each piece in which one begins and 256 columns.  Its waves
// take kJoin parts each in turn, then the first adds the others' sums in order.
constexpr int kJoin = 16, kJoinWaves = 4;
template <bool SUMS>
__global__ __launch_bounds__(64 * kJoinWaves) void k_embed_join(const EmbedGrad a) {
  __shared__ float sums[kJoinWaves - 1][4][64];
  const int lane = threadIdx.x & (kWave - 1), w = threadIdx.x / kWave, D = a.D;
  const int64_t p = blockIdx.x;
  const int64_t s0 = p * a.len, s1 = s0 + a.len;      // (the last piece begins none that is cut)
  const uint32_t k = a.key_at(s1 - 1), k_next = a.key_at(s1), k0 = a.key_at(s0);
  const uint32_t k_prev = s0 > 0 ? a.key_at(s0 - 1) : (uint32_t)a.V + 1;
  if (k == (uint32_t)a.V || k_next != k) return;   // nothing goes on behind this piece
  if (k0 == k && k_prev == k) return;              // the run began before it
  // pieces that the run goes on in: the next one, and every one that starts with it
  int64_t more = 1;
  for (;;) {
    const int64_t q = p + 1 + more + lane;
    const bool on = q < a.pieces && a.key_at(q * a.len) == k;
    const uint64_t m = __ballot(on);
    more += m == ~0ull ? 64 : __builtin_ctzll(~m);
    if (m != ~0ull) break;
  }
  const int ct = ((int)blockIdx.y * kWave + lane) * 4, c = ct < D ? run_start<4>(ct, D) : D, n = D - c;
  float acc[4] = {0.0f, 0.0f, 0.0f, 0.0f};
  if (w == 0) load_some<4>(a.part, false, (p * 2 + 1) * D + c, n, acc);
  for (int64_t q0 = 1 + w * kJoin; q0 <= more; q0 += kJoinWaves * kJoin) {
    float v[kJoin][4];
#pragma unroll
    for (int u = 0; u < kJoin; ++u)
      if (q0 + u <= more) load_some<4>(a.part, false, (p + q0 + u) * 2 * D + c, n, v[u]);
#pragma unroll
    for (int u = 0; u < kJoin; ++u)
      if (q0 + u <= more) {
#pragma unroll
        for (int j = 0; j < 4; ++j) acc[j] += v[u][j];
      }
  }
  if (more > kJoin) {   // (else the others have nothing)
    if (w > 0) {
#pragma unroll
      for (int j = 0; j < 4; ++j) sums[w - 1][j][lane] = acc[j];
    }
    __syncthreads();
    if (w == 0) {
#pragma unroll
      for (int g = 0; g < kJoinWaves - 1; ++g)
#pragma unroll
        for (int j = 0; j < 4; ++j) acc[j] += sums[g][j][lane];
    }
  }
  int64_t at = k;
  if (SUMS) {   // the run's first pair
    int64_t lo = s0, hi = s1 - 1;
    while (lo < hi) {
      const int64_t mid = (lo + hi) >> 1;
      if (a.key_at(mid) < k)
        lo = mid + 1;
      else
        hi = mid;
    }
    at = lo;
  }
  if (w == 0) embed_store<4>(a, at * D + c, n, acc);
}

static bool embed_type(int dtype) { return dtype == NSA_F32 || dtype == NSA_BF16; }

// Pairs a thread of the sort (4, more past 256 blocks), and its blocks
static int sort_per(int64_t n) {
  const int64_t per = (n + kSortThreads * 256 - 1) / (kSortThreads * 256);
  return (int)((per + kSortAhead - 1) / kSortAhead * kSortAhead);
}
static int sort_blocks(int64_t n) {
  const int64_t per = (int64_t)kSortThreads * sort_per(n);
  return (int)((n + per - 1) / per);
}
// Pairs a piece: 8, more where the pieces would be more than 2048
static int embed_piece(int64_t n, int most = 2048) {
  int64_t len = 8;
  while (n / len > most) len *= 2;
  return (int)len;
}
struct EmbedPlan {
  int64_t pairs;         // of one buffer, rounded up to 16 bytes
  int64_t counts, parts;
  int len, pieces;
  size_t bytes() const { return (size_t)(4 * pairs + counts + parts) * 4; }
};
static EmbedPlan embed_plan(int64_t n, int D, bool sorted, int most = 2048) {
  EmbedPlan p;
  p.pairs = sorted ? (n + 3) / 4 * 4 : 0;
  p.counts = sorted ? sort_blocks(n) * kSortBins : 0;
  p.len = embed_piece(n, most);
  p.pieces = (int)((n + p.len - 1) / p.len);
  p.parts = (int64_t)p.pieces * 2 * D;
  return p;
}

// The workspace of such a plan: two buffers of pairs in turn, the sort's counts, the runs' parts.
struct EmbedLists {
  uint32_t *key, *val, *key2, *val2, *count;
  float* part;
  EmbedLists(void* ws, const EmbedPlan& p)
      : key(static_cast<uint32_t*>(ws)),
        val(key + p.pairs),
        key2(val + p.pairs),
        val2(key2 + p.pairs),
        count(val2 + p.pairs),
        part(reinterpret_cast<float*>(count + p.counts)) {}
};

// (index, i) sorted into key and val
static void embed_sort(EmbedLists& at, const int64_t* index, int64_t n, int64_t V, hipStream_t s) {
  int bits = 1;   // of the keys 0 .. V
  while ((V >> bits) != 0) ++bits;
  const int passes = (bits + kSortBits - 1) / kSortBits;
  if (n <= kSmallSort) {
    k_sort_small<<<1, 1024, 0, s>>>(index, at.key, at.val, (int)n, V, passes, bits);
    return;
  }
  const unsigned blocks = (unsigned)sort_blocks(n);
  for (int q = 0, shift = 0; q < passes; ++q) {
    const int b = (bits - shift + passes - q - 1) / (passes - q);
    const SortPass a{q == 0 ? index : nullptr, at.key, at.val, at.key2, at.val2, at.count, n, V, sort_per(n), shift, b};
    k_sort_count<<<blocks, kSortThreads, 0, s>>>(a);
    k_sort_move<<<blocks, kSortThreads, 0, s>>>(a);
    shift += b;
    std::swap(at.key, at.key2);
    std::swap(at.val, at.val2);
  }
}

template <int E, bool SUMS>
static void embed_sums(const EmbedGrad& g, bool join, hipStream_t s) {
  const int64_t clear = (g.V + 63) / 64;
  const unsigned grid = (unsigned)(g.pieces + (clear < (1 << 16) ? clear : 1 << 16));
  const int runs = (g.D + E - 1) / E, nth = runs >= 256 ? 256 : (runs + 63) / 64 * 64;
  k_embed_runs<E, SUMS><<<dim3(grid, (unsigned)((runs + nth - 1) / nth)), nth, 0, s>>>(g);
  if (g.pieces > 1 && join)
    k_embed_join<SUMS><<<dim3((unsigned)(g.pieces - 1), (unsigned)((g.D + 255) / 256)), 64 * kJoinWaves, 0, s>>>(g);
}

}  // namespace nsa

extern "C" int nsa_embed_fwd(const int64_t* tokens, const int64_t* pos, const void* w, const void* pw, void* out,
                             int64_t n, int64_t T, int64_t V, int64_t P, int D, float scale, int w_dtype, int pw_dtype,
                             int out_dtype, void* stream) {
  using namespace nsa;
  NSA_CHECK(n >= 0 && n <= kEmbedRows && V >= 1 && V <= kEmbedRows && D >= 1 && D <= kEmbedWide, NSA_ERR_SHAPE);
  NSA_CHECK(embed_type(w_dtype) && embed_type(out_dtype), NSA_ERR_DTYPE);
  if (pw != nullptr) {
    NSA_CHECK(P >= 1 && P <= kEmbedRows && (n == 0 || pos != nullptr || (T >= 1 && T <= kEmbedRows)), NSA_ERR_SHAPE);
    NSA_CHECK(embed_type(pw_dtype), NSA_ERR_DTYPE);
  }
  if (n == 0) return NSA_OK;
  NSA_CHECK(tokens != nullptr && w != nullptr && out != nullptr, NSA_ERR_ARG);
  const hipStream_t s = static_cast<hipStream_t>(stream);
  // 2^24 rows a launch: a grid holds less than 2^32 threads
  for (int64_t r0 = 0; r0 < n; r0 += 1 << 24) {
    const int64_t end = n - r0 < (1 << 24) ? n : r0 + (1 << 24);
    // an output that the caches cannot hold leaves them to the tables (8 x 4096 rows of 768
    // in float32: 37 us, 42 through the caches)
    const bool past = (double)n * D * (out_dtype == NSA_BF16 ? 2 : 4) > (double)(64 << 20);
    const EmbedArgs a{tokens, pos, w, pw, out, r0, end, T, V, P, D, scale, w_dtype == NSA_BF16, pw_dtype == NSA_BF16,
                      out_dtype == NSA_BF16};
    auto go = [&](auto e, auto tpr) {
      constexpr int E = decltype(e)::value, TPR = decltype(tpr)::value;
      const unsigned grid = (unsigned)((end - r0 + 256 / TPR - 1) / (256 / TPR));
      if (past)
        k_embed_fwd<E, TPR, true><<<grid, 256, 0, s>>>(a);
      else
        k_embed_fwd<E, TPR, false><<<grid, 256, 0, s>>>(a);
    };
    // the fewest threads that hold a row with 16 elements each, 64 at most
    auto pick = [&](auto e) {
      if (D <= 64)
        go(e, std::integral_constant<int, 4>{});
      else if (D <= 256)
        go(e, std::integral_constant<int, 16>{});
      else
        go(e, std::integral_constant<int, 64>{});
    };
    if (w_dtype == NSA_BF16)
      pick(std::integral_constant<int, 8>{});
    else
      pick(std::integral_constant<int, 4>{});
    const int rc = nsa_launch_status();
    if (rc != NSA_OK) return rc;
  }
  return NSA_OK;
}

extern "C" size_t nsa_embed_bwd_workspace(int64_t n, int D, int sorted) {
  using namespace nsa;
  if (n < 0 || n > kEmbedRows || D < 1 || D > kEmbedWide) return 0;
  if (n == 0) return 16;
  return embed_plan(n, D, sorted != 0).bytes();
}

extern "C" int nsa_embed_bwd(const int64_t* index, const void* dy, void* dw, void* workspace, size_t workspace_bytes,
                             int64_t n, int64_t T, int64_t V, int D, float scale, int dy_dtype, int w_dtype,
                             void* stream) {
  using namespace nsa;
  NSA_CHECK(n >= 1 && n <= kEmbedRows && V >= 1 && V <= kEmbedRows && D >= 1 && D <= kEmbedWide, NSA_ERR_SHAPE);
  NSA_CHECK(index != nullptr || (T >= 1 && T <= V && n % T == 0), NSA_ERR_SHAPE);
  NSA_CHECK(embed_type(dy_dtype) && embed_type(w_dtype), NSA_ERR_DTYPE);
  NSA_CHECK(dy != nullptr && dw != nullptr, NSA_ERR_ARG);
  const EmbedPlan p = embed_plan(n, D, index != nullptr);
  NSA_CHECK(workspace != nullptr && workspace_bytes >= p.bytes(), NSA_ERR_WORKSPACE);
  NSA_CHECK(reinterpret_cast<uintptr_t>(workspace) % 16 == 0, NSA_ERR_ARG);
  const hipStream_t s = static_cast<hipStream_t>(stream);
  EmbedLists at(workspace, p);
  if (index != nullptr) embed_sort(at, index, n, V, s);
  // positions 0 .. T-1 of up to 64 sequences: whole runs a piece, none to join
  const int64_t B = index != nullptr ? 1 : n / T;
  const bool whole = index == nullptr && B <= 64;
  const int len = whole ? (int)((p.len + B - 1) / B * B) : p.len, pieces = (int)((n + len - 1) / len);
  const EmbedGrad g{index != nullptr ? at.key : nullptr, at.val, dy, dw, at.part, n, T, V, (uint32_t)B,
                    D, len, pieces, scale, dy_dtype == NSA_BF16, w_dtype == NSA_BF16, nullptr, nullptr, nullptr};
  if (g.dy_bf16)
    embed_sums<8, false>(g, !whole, s);
  else
    embed_sums<4, false>(g, !whole, s);
  return nsa_launch_status();
}

// (fewer and longer pieces of wide rows, which several workgroups share: 8192 x 4096 in 40 us,
// 52 with 1024 pieces; 32768 x 768 in 31 with 2048, 59 with 512)
static nsa::EmbedPlan token_sums_plan(int64_t n, int D) { return nsa::embed_plan(n, D, true, D > 2048 ? 512 : 2048); }

size_t nsa_token_sums_workspace(int64_t n, int D) { return token_sums_plan(n, D).bytes(); }

int nsa_token_sums(const int64_t* index, const float* weight, const void* rows, void* sums, int* first, uint64_t* there,
                   void* workspace, int64_t n, int64_t V, int D, void* stream) {
  using namespace nsa;
  const hipStream_t s = static_cast<hipStream_t>(stream);
  const EmbedPlan p = token_sums_plan(n, D);
  EmbedLists at(workspace, p);
  embed_sort(at, index, n, V, s);
  const EmbedGrad g{at.key, at.val, rows,     sums, at.part, n,    1,      V,     1,
                    D,      p.len,  p.pieces, 1.0f, true,    true, weight, first, there};
  embed_sums<8, true>(g, true, s);
  return nsa_launch_status();
}
