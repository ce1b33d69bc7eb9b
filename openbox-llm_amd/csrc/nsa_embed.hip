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
//      pairs; places from the counts, ranks within a wave by ballots).  Positions
//      0 .. T-1 of every sequence need no sort: the sorted list is a formula.
//   2. The sorted list is cut into pieces of equal length, whatever the tokens'
//      frequencies (in text one token can be a tenth of all): a workgroup adds the
//      rows of its piece one after another and writes a token's row where the run
//      of the token ends.  A run that is cut leaves its parts in float32.  Other
//      workgroups of the same launch clear the rows without a token, so that the
//      table is written once.
//   3. The parts of every cut run are added in the order of the pieces.
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

// TPR threads a row, 256 / TPR rows a workgroup.
template <int TPR>
__global__ __launch_bounds__(256) void k_embed_fwd(const EmbedArgs a) {
  const int t = threadIdx.x & (TPR - 1);
  const int64_t i = a.first + (int64_t)blockIdx.x * (256 / TPR) + threadIdx.x / TPR;
  if (i >= a.n) return;
  const int64_t tok = a.tokens[i];
  const bool real = tok >= 0 && tok < a.V;
  const int64_t p = a.pw == nullptr ? 0 : a.pos != nullptr ? a.pos[i] : i % a.T;
  const bool has_pos = a.pw != nullptr && p >= 0 && p < a.P;
  const int D = a.D;
#pragma unroll 2
  for (int c = 8 * t; c < D; c += 8 * TPR) {
    const int n = D - c;
    float v[8] = {0, 0, 0, 0, 0, 0, 0, 0}, q[8] = {0, 0, 0, 0, 0, 0, 0, 0};
    if (real) load_run8_of(a.w, a.w_bf16, tok * D + c, n, v);
    if (has_pos) load_run8_of(a.pw, a.pw_bf16, p * D + c, n, q);
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = real ? fmaf(v[j], a.scale, q[j]) : q[j];
    if (a.out_bf16)
      store_run8(static_cast<bf16*>(a.out) + i * D + c, n, v);
    else
      store_run8(static_cast<float*>(a.out) + i * D + c, n, v);
  }
}

// ---------------------------------------------------------------------------
// sort of (key, i) by key, ties by i
// ---------------------------------------------------------------------------
constexpr int kSortThreads = 256;
constexpr int kSortWaves = kSortThreads / kWave;
constexpr int kSortBits = 9;
constexpr int kSortBins = 1 << kSortBits;

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
  for (int r = 0; r < a.per; ++r) {
    const int64_t i = first + (int64_t)r * kSortThreads + threadIdx.x;
    if (i < a.n) atomicAdd(&bins[(sort_key(a, i) >> a.shift) & (nb - 1)], 1u);
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
  // places of the block's digits: all smaller digits, then this digit's earlier blocks
  constexpr int kPer = kSortBins / kSortThreads;
  uint32_t total[kPer], before[kPer], mine = 0;
#pragma unroll
  for (int k = 0; k < kPer; ++k) {
    const int b = tid * kPer + k;
    total[k] = before[k] = 0;
    if (b < nb) {
#pragma unroll 8
      for (int g = 0; g < (int)gridDim.x; ++g) {
        const uint32_t c = a.count[(int64_t)g * nb + b];
        total[k] += c;
        before[k] += g < (int)blockIdx.x ? c : 0u;
      }
    }
    mine += total[k];
  }
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
  const int64_t first = (int64_t)blockIdx.x * kSortThreads * a.per + (int64_t)w * kWave * a.per;
  // 1st walk: how many pairs of each digit every wave has
  for (int r = 0; r < a.per; ++r) {
    const int64_t i = first + (int64_t)r * kWave + lane;
    if (i < a.n) atomicAdd(&seen[w][(sort_key(a, i) >> a.shift) & (nb - 1)], 1u);
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
  for (int r = 0; r < a.per; ++r) {
    const int64_t i = first + (int64_t)r * kWave + lane;
    const bool ok = i < a.n;
    const uint32_t key = ok ? sort_key(a, i) : 0u;
    const uint32_t dig = (key >> a.shift) & (nb - 1);
    uint64_t same = __ballot(ok);
    for (int b = 0; b < a.bits; ++b) {
      const uint64_t m = __ballot((dig >> b) & 1u);
      same &= (dig >> b) & 1u ? m : ~m;
    }
    if (ok) {
      const uint32_t rank = (uint32_t)__popcll(same & ((1ull << lane) - 1ull));
      const uint32_t to = seen[w][dig] + rank;
      a.key_out[to] = key;
      a.val_out[to] = a.tokens != nullptr ? (uint32_t)i : a.val_in[i];
    }
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");   // (LDS accesses of a wave keep their order: all have read before one adds)
    if (ok && (same >> lane) == 1ull) seen[w][dig] += (uint32_t)__popcll(same);
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  }
}

// ---------------------------------------------------------------------------
// sums over the runs of the sorted list
// ---------------------------------------------------------------------------
constexpr int kAhead = 4;   // rows asked for at a time

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
  // (fewer than 2^31 pairs: 32-bit divisions)
  __device__ __forceinline__ uint32_t key_at(int64_t s) const { return key != nullptr ? key[s] : (uint32_t)s / B; }
  __device__ __forceinline__ int64_t row_at(int64_t s) const {
    return key != nullptr ? (int64_t)val[s] : (int64_t)((uint32_t)s % B) * T + (uint32_t)s / B;
  }
};

__device__ __forceinline__ void embed_store(const EmbedGrad& a, int64_t at, int n, const float (&v)[8]) {
  float o[8];
#pragma unroll
  for (int j = 0; j < 8; ++j) o[j] = v[j] * a.scale;
  if (a.w_bf16)
    store_run8(static_cast<bf16*>(a.dw) + at, n, o);
  else
    store_run8(static_cast<float*>(a.dw) + at, n, o);
}

// Clear the rows r0 .. r0 + 63 that have no token.
template <int NTH>
__device__ __forceinline__ void embed_clear(const EmbedGrad& a, int64_t r0) {
  const int tid = threadIdx.x, D = a.D;
  const int64_t v = r0 + (tid & 63);
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
  }
  uint64_t rows = __ballot(empty);   // (every wave of the workgroup: the same)
  const float zero[8] = {0, 0, 0, 0, 0, 0, 0, 0};
  while (rows != 0) {
    const int64_t at = (r0 + __builtin_ctzll(rows)) * D;
    rows &= rows - 1;
    for (int c = 8 * tid; c < D; c += 8 * NTH) {
      if (a.w_bf16)
        store_run8(static_cast<bf16*>(a.dw) + at + c, D - c, zero);
      else
        store_run8(static_cast<float*>(a.dw) + at + c, D - c, zero);
    }
  }
}

// Workgroups below a.pieces add the rows of a piece; the others clear the rows
// without a token, 64 rows of the table at a time.  A thread owns runs of 8 columns.
template <int NTH>
__global__ __launch_bounds__(NTH) void k_embed_runs(const EmbedGrad a) {
  const int tid = threadIdx.x, D = a.D;
  if ((int)blockIdx.x >= a.pieces) {
    for (int64_t r0 = ((int64_t)blockIdx.x - a.pieces) * 64; r0 < a.V; r0 += ((int64_t)gridDim.x - a.pieces) * 64)
      embed_clear<NTH>(a, r0);
    return;
  }
  const int64_t s0 = (int64_t)blockIdx.x * a.len, s1 = s0 + a.len < a.n ? s0 + a.len : a.n;
  const uint32_t none = (uint32_t)a.V;
  const uint32_t k_prev = s0 > 0 ? a.key_at(s0 - 1) : none + 1, k_next = s1 < a.n ? a.key_at(s1) : none + 1;
  float* part = a.part + (int64_t)blockIdx.x * 2 * D;
  for (int c = 8 * tid; c < D; c += 8 * NTH) {
    const int n = D - c;
    float acc[8] = {0, 0, 0, 0, 0, 0, 0, 0};
    uint32_t k = a.key_at(s0);
    bool head = k == k_prev;   // the run began in an earlier piece
    for (int64_t s = s0; s < s1 && k != none; s += kAhead) {
      float v[kAhead][8];
      uint32_t kn[kAhead];     // the key behind each row (none + 1 behind the piece)
#pragma unroll
      for (int u = 0; u < kAhead; ++u) {
        if (s + u < s1) load_run8_of(a.dy, a.dy_bf16, a.row_at(s + u) * D + c, n, v[u]);
        kn[u] = s + u + 1 < s1 ? a.key_at(s + u + 1) : none + 1;
      }
#pragma unroll
      for (int u = 0; u < kAhead; ++u) {
        if (s + u >= s1 || k == none) continue;
#pragma unroll
        for (int j = 0; j < 8; ++j) acc[j] += v[u][j];
        if (kn[u] == k) continue;
        if (head)
          store_run8(part + c, n, acc);
        else if (s + u + 1 == s1 && k == k_next)   // the run goes on in the next piece
          store_run8(part + D + c, n, acc);
        else
          embed_store(a, (int64_t)k * D + c, n, acc);
        head = false;
        k = kn[u];
#pragma unroll
        for (int j = 0; j < 8; ++j) acc[j] = 0.0f;
      }
    }
  }
}

// The cut runs: one workgroup for each piece in which one begins.
template <int NTH>
__global__ __launch_bounds__(NTH) void k_embed_join(const EmbedGrad a) {
  const int tid = threadIdx.x, lane = tid & (kWave - 1), D = a.D;
  const int64_t p = blockIdx.x;
  const int64_t s0 = p * a.len, s1 = s0 + a.len;      // (the last piece begins none that is cut)
  const uint32_t k = a.key_at(s1 - 1);
  if (k == (uint32_t)a.V || a.key_at(s1) != k) return;               // nothing goes on behind this piece
  if (a.key_at(s0) == k && s0 > 0 && a.key_at(s0 - 1) == k) return;  // the run began before it
  // pieces that the run goes on in: the next one, and every one that starts with it
  int64_t more = 1;
  for (;;) {
    const int64_t q = p + 1 + more + lane;
    const bool on = q < a.pieces && a.key_at(q * a.len) == k;
    const uint64_t m = __ballot(on);
    more += m == ~0ull ? 64 : __builtin_ctzll(~m);
    if (m != ~0ull) break;
  }
  for (int c = 8 * tid; c < D; c += 8 * NTH) {
    const int n = D - c;
    float acc[8];
    load_run8(a.part + (p * 2 + 1) * D + c, n, acc);
#pragma unroll 4
    for (int64_t q = 1; q <= more; ++q) {
      float v[8];
      load_run8(a.part + (p + q) * 2 * D + c, n, v);
#pragma unroll
      for (int j = 0; j < 8; ++j) acc[j] += v[j];
    }
    embed_store(a, (int64_t)k * D + c, n, acc);
  }
}

static bool embed_type(int dtype) { return dtype == NSA_F32 || dtype == NSA_BF16; }

// Pairs a thread of the sort (4, more past 256 blocks), and its blocks
static int sort_per(int64_t n) {
  const int64_t per = (n + kSortThreads * 256 - 1) / (kSortThreads * 256);
  return per < 4 ? 4 : (int)per;
}
static int sort_blocks(int64_t n) {
  const int64_t per = (int64_t)kSortThreads * sort_per(n);
  return (int)((n + per - 1) / per);
}
// Pairs a piece: 32, more where the pieces would be more than 4096
static int embed_piece(int64_t n) {
  int64_t len = 32;
  while (n / len > 4096) len *= 2;
  return (int)len;
}
struct EmbedPlan {
  int64_t pairs;         // of one buffer, rounded up to 16 bytes
  int64_t counts, parts;
  int len, pieces;
  size_t bytes() const { return (size_t)(4 * pairs + counts + parts) * 4; }
};
static EmbedPlan embed_plan(int64_t n, int D, bool sorted) {
  EmbedPlan p;
  p.pairs = sorted ? (n + 3) / 4 * 4 : 0;
  p.counts = sorted ? sort_blocks(n) * kSortBins : 0;
  p.len = embed_piece(n);
  p.pieces = (int)((n + p.len - 1) / p.len);
  p.parts = (int64_t)p.pieces * 2 * D;
  return p;
}

}  // namespace nsa

extern "C" int nsa_embed_fwd(const int64_t* tokens, const int64_t* pos, const void* w, const void* pw, void* out,
                             int64_t n, int64_t T, int64_t V, int64_t P, int D, float scale, int w_dtype, int pw_dtype,
                             int out_dtype, void* stream) {
  using namespace nsa;
  NSA_CHECK(n >= 0 && n <= kEmbedRows && V >= 1 && V <= kEmbedRows && D >= 1 && D <= kEmbedWide, NSA_ERR_SHAPE);
  NSA_CHECK(embed_type(w_dtype) && embed_type(out_dtype), NSA_ERR_DTYPE);
  if (pw != nullptr) {
    NSA_CHECK(P >= 1 && P <= kEmbedRows && (pos != nullptr || T >= 1), NSA_ERR_SHAPE);
    NSA_CHECK(embed_type(pw_dtype), NSA_ERR_DTYPE);
  }
  if (n == 0) return NSA_OK;
  NSA_CHECK(tokens != nullptr && w != nullptr && out != nullptr, NSA_ERR_ARG);
  const hipStream_t s = static_cast<hipStream_t>(stream);
  const int runs = (D + 7) / 8;
  // 2^24 rows a launch: a grid holds less than 2^32 threads
  for (int64_t r0 = 0; r0 < n; r0 += 1 << 24) {
    const int64_t end = n - r0 < (1 << 24) ? n : r0 + (1 << 24);
    const EmbedArgs a{tokens, pos, w, pw, out, r0, end, T, V, P, D, scale, w_dtype == NSA_BF16, pw_dtype == NSA_BF16,
                      out_dtype == NSA_BF16};
    auto grid = [&](int tpr) { return (unsigned)((end - r0 + 256 / tpr - 1) / (256 / tpr)); };
    // the fewest threads that hold a row with one run each, 64 at most
    if (runs <= 4)
      k_embed_fwd<4><<<grid(4), 256, 0, s>>>(a);
    else if (runs <= 16)
      k_embed_fwd<16><<<grid(16), 256, 0, s>>>(a);
    else if (runs <= 32)
      k_embed_fwd<32><<<grid(32), 256, 0, s>>>(a);
    else
      k_embed_fwd<64><<<grid(64), 256, 0, s>>>(a);
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
  const hipStream_t s = static_cast<hipStream_t>(stream);
  uint32_t* ws = static_cast<uint32_t*>(workspace);
  uint32_t *ka = ws, *va = ka + p.pairs, *kb = va + p.pairs, *vb = kb + p.pairs, *count = vb + p.pairs;
  float* part = reinterpret_cast<float*>(count + p.counts);
  if (index != nullptr) {
    int bits = 1;   // of the keys 0 .. V
    while ((V >> bits) != 0) ++bits;
    const int passes = (bits + kSortBits - 1) / kSortBits;
    const unsigned blocks = (unsigned)sort_blocks(n);
    for (int q = 0, shift = 0; q < passes; ++q) {
      const int b = (bits - shift + passes - q - 1) / (passes - q);
      const SortPass a{q == 0 ? index : nullptr, ka, va, kb, vb, count, n, V, sort_per(n), shift, b};
      k_sort_count<<<blocks, kSortThreads, 0, s>>>(a);
      k_sort_move<<<blocks, kSortThreads, 0, s>>>(a);
      shift += b;
      uint32_t* t = ka;
      ka = kb, kb = t;
      t = va;
      va = vb, vb = t;
    }
  }
  const EmbedGrad g{index != nullptr ? ka : nullptr, va, dy, dw, part, n, T, V, (uint32_t)(index != nullptr ? 1 : n / T),
                    D, p.len, p.pieces, scale, dy_dtype == NSA_BF16, w_dtype == NSA_BF16};
  const int64_t clear = (V + 63) / 64;
  const unsigned grid = (unsigned)(p.pieces + (clear < (1 << 16) ? clear : 1 << 16));
  auto go = [&](auto nth) {
    constexpr int N = decltype(nth)::value;
    k_embed_runs<N><<<grid, N, 0, s>>>(g);
    if (p.pieces > 1) k_embed_join<N><<<(unsigned)(p.pieces - 1), N, 0, s>>>(g);
  };
  // threads that hold a row with one run each, 256 at most
  if (D <= 512)
    go(std::integral_constant<int, 64>{});
  else if (D <= 1024)
    go(std::integral_constant<int, 128>{});
  else
    go(std::integral_constant<int, 256>{});
  return nsa_launch_status();
}
