// Log probabilities of given tokens, the entropy and the best alternatives of
// every row of logits z [rows][V], in one pass over the row, and the gradient.
//
//   m = max z,  l = sum e^(z-m),  s = sum e^(z-m) (z-m)
//   logp = (z_t - m) - ln l,   H = ln l - s / l,   top: z descending, index ascending
//   dz_j = dlogp (1[j = t] - p_j) - dH p_j (ln p_j + H),   p_j = e^(z_j - m) / l
//
// m is the row's own maximum, never a sentinel: it starts at the lowest finite
// value, so that minus infinity has weight 0 against it (e^-inf) while a row
// masked with the type's lowest value still sums to its length.  NaN and plus
// infinity make l NaN, and with it the row's results.
//
// The forward reads the row once.  A lane keeps its own (m, l, s) and rescales
// them when its runs of a chunk raise its maximum.  For the alternatives the k-th
// largest of 64 or 256 maxima over parts of the row is a lower bound of the
// row's k-th value (k parts hold one such element each).  It is formed after the
// first chunk and again whenever the chunks done are four times as many: 16
// ballots, one for each of the upper bits of a value's key.  Runs with nothing at
// or above it are dropped; the others are noted, and at the end read again, all
// at once: the loop waits for no load but its own.  Their elements (24 of 32000
// for 20 alternatives) go to a list in LDS as (value, ~index) keys, which are all
// different, and are ranked by counting.  Masked elements (-inf, the type's
// lowest value) are never noted.  A row that overfills a list (long ties, a
// rising row), or that has fewer than k unmasked elements, is selected exactly
// by up to eight radix passes over the keys instead (32 x 32000 with five tokens
// left and 20 alternatives: 50 us; 238 with every lane's own LDS atomics and all
// eight passes).
//
// Measured (MI355X): 32768 x 32000 in bf16 384 us forward and 737 backward, 5.5
// and 5.7 TB/s, bound by memory; 2047 x 50257 45 us, 49 with 5 and 50 with 20
// alternatives in a captured loop (38 at the rate of a large copy: all rows are
// resident at once, so that they start and end together); 32 x 32000 with 20 8.5
// us, a row's own chain of load, sums, bound and ranking.
//
// A weight e^x, x = z - m, is formed as 2^(x log2 e): the product's rounding makes
// it right to about |x| 2^-24, so that the lighter a weight the less exact it is.
//
// One wave takes a row of up to 2048 elements (8192 where the rows are many), a
// workgroup of four or sixteen a longer one; few and very long rows are split over
// workgroups, whose (m, l, s) and lists a second launch joins.
#include <type_traits>

#include "nsa_launch.h"
#include "nsa_rows.h"

namespace nsa {

constexpr int kLpTopMax = 64;        // most alternatives
constexpr int kLpCap = 1024;         // candidate list
constexpr int64_t kLpSlice = 1 << 21;   // rows of one launch
constexpr float kLowest = -3.402823466e38f;
constexpr float kFar = -1.0e30f;     // stands for the logarithm of weight 0 where it is multiplied by 0

struct LpArgs {
  const void* z;
  const int64_t* target;   // or null
  float *logp, *entropy;
  float2* stat;            // (m, ln l); or null
  float* top_logp;         // [rows][k]
  int64_t* top_idx;
  float4* part;            // [rows][nsp] (m, l, s) of a split row
  uint64_t* part_top;      // [rows][nsp][k] keys, descending, 0 past the part's elements
  int64_t rows;
  int V, k, nsp, seg;      // parts a row, elements a part
};

// z's key: the order of the values, -0 with 0, NaN above infinity; ties to the lower index
__device__ __forceinline__ uint32_t value_key(float z) {
  return z != z ? 0xffffffffu : order_key(z + 0.0f);
}
__device__ __forceinline__ uint64_t elem_key(float z, int idx) {
  return ((uint64_t)value_key(z) << 32) | (uint32_t)~idx;
}
__device__ __forceinline__ float key_value(uint64_t key) {
  const uint32_t u = (uint32_t)(key >> 32);
  return __uint_as_float((u & 0x80000000u) ? (u ^ 0x80000000u) : ~u);
}

struct LpState {
  float m, l, s;
};
__device__ __forceinline__ void lp_raise(LpState& a, float m) {   // a's sums against the maximum m >= a.m
  const float d = a.m - m;
  const float f = fast_exp2(d * kLog2e);
  a.l *= f;
  a.s = a.s * f + a.l * fmaxf(d, kFar);
  a.m = m;
}
// The sums of W waves (W > 1: two barriers, buf is free before and after):
// the common maximum first, so that every lane rescales once.
template <int W>
__device__ __forceinline__ LpState lp_group(LpState a, float (&buf)[3][W]) {
  const int w = threadIdx.x >> 6;
  const bool first = (threadIdx.x & 63) == 0;
  float m = wave_max(a.m);
  if (W > 1) {
    if (first) buf[0][w] = m;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < W; ++i) m = fmaxf(m, buf[0][i]);
  }
  lp_raise(a, m);
  a.l = wave_sum(a.l);
  a.s = wave_sum(a.s);
  if (W > 1) {
    if (first) buf[1][w] = a.l, buf[2][w] = a.s;
    __syncthreads();
    a.l = a.s = 0.0f;
#pragma unroll
    for (int i = 0; i < W; ++i) a.l += buf[1][i], a.s += buf[2][i];
  }
  return a;
}

// Results of one row from its sums (one thread).
__device__ __forceinline__ void lp_finish(const LpArgs& a, int64_t row, LpState st, float zt, bool has_t) {
  const float logl = st.l == 0.0f ? -__builtin_inff() : logf(st.l);
  if (a.stat != nullptr) a.stat[row] = make_float2(st.m, logl);
  if (a.entropy != nullptr) a.entropy[row] = st.l == 0.0f ? 0.0f : logl - st.s / st.l;
  if (a.logp != nullptr) a.logp[row] = has_t ? (st.l == 0.0f ? -__builtin_inff() : (zt - st.m) - logl) : 0.0f;
}

// The target's logit: asked for at the start, so that its load is not waited for at the end.
template <typename T>
__device__ __forceinline__ bool lp_target(const LpArgs& a, int64_t row, float& zt) {
  if (a.target == nullptr) return false;
  const int64_t t = a.target[row];
  if (t < 0 || t >= a.V) return false;
  zt = (float)static_cast<const T*>(a.z)[row * a.V + t];
  return true;
}

// The k best of the `count` keys in LDS, by rank: THR threads; place[rank] = key
template <int THR, typename F>
__device__ __forceinline__ void lp_rank(const uint64_t* list, int count, int k, int t, F place) {
  for (int i = t; i < count; i += THR) {
    const uint64_t mine = list[i];
    int rank = 0;
    for (int j = 0; j < count; ++j) rank += list[j] > mine ? 1 : 0;
    if (rank < k) place(rank, mine);
  }
}

// The k-th largest of 16-bit values, N a lane: bit by bit from the top.
template <int N>
__device__ __forceinline__ uint32_t lp_kth(const uint32_t (&v)[N], int k) {
  uint32_t kth = 0;
#pragma unroll
  for (int bit = 15; bit >= 0; --bit) {
    const uint32_t cand = kth | (1u << bit);
    int n = 0;
#pragma unroll
    for (int i = 0; i < N; ++i) n += __popcll(__ballot(v[i] >= cand));
    kth = n >= k ? cand : kth;
  }
  return kth;
}

// The lowest finite value of a type's key.
template <typename T>
__device__ constexpr uint32_t lowest_key() {
  return sizeof(T) == 2 ? 0x0080ffffu : 0x00800000u;   // ~0xff7f0000, ~0xff7fffff
}

// W waves a row (1: four rows a workgroup of 256 threads); U runs of 8 a lane and chunk.
template <typename T, int W, int U, bool TOP>
__global__ __launch_bounds__(W > 4 ? 64 * W : 256, W > 4 ? 4 : 8) void k_logprob(const LpArgs a) {
  constexpr int THR = 64 * W;               // threads a row
  constexpr int ROWS = W > 1 ? 1 : 4;       // rows a workgroup
  constexpr int CAP = W > 1 ? kLpCap : 512;
  constexpr int RUNS = W > 1 ? kLpCap : 256;   // list of runs, in the place of the radix passes' counts
  __shared__ uint64_t list_s[TOP ? ROWS : 1][TOP ? CAP : 1];
  __shared__ uint32_t keys_s[2][TOP && W > 1 ? THR : 1];
  __shared__ __align__(16) uint32_t hist[TOP ? ROWS : 1][TOP ? RUNS : 1];
  __shared__ int nruns_s[ROWS], count_s[ROWS];
  __shared__ float st_s[3][W];
  const int t = threadIdx.x & (THR - 1), sub = threadIdx.x / THR;
  const int64_t unit = (int64_t)blockIdx.x * ROWS + sub;
  const int64_t row = ROWS > 1 ? unit : unit / a.nsp;
  const int part = ROWS > 1 ? 0 : (int)(unit % a.nsp);
  const bool live = row < a.rows;           // (whole waves; the barriers below are for every wave)
  const int c0 = part * a.seg;
  const int c1 = live ? min(a.V, c0 + a.seg) : c0;
  const T* z = static_cast<const T*>(a.z) + (live ? row : 0) * a.V;
  float zt = 0.0f;
  const bool has_t = live && t == 0 && lp_target<T>(a, row, zt);
  uint64_t* list = list_s[TOP ? sub : 0];
  auto sync = [] {
    if (W > 1)
      __syncthreads();
    else
      __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  };
  if (TOP && t == 0) nruns_s[sub] = count_s[sub] = 0;   // (added to only behind the first bound's barrier)

  LpState st{kLowest, 0.0f, 0.0f};
  constexpr uint32_t kMasked = lowest_key<T>();
  uint32_t thr = kMasked + 1;   // keys below it are no alternatives: masked elements least of all
  float thr_z = key_value((uint64_t)thr << 32);
  int next = 1;                 // chunks done at the bound's next forming
  int done = 0, turn = 0;
  constexpr int CH = THR * 8 * U;
  // runs start at 16-byte addresses, the first one up to 7 elements before c0: odd rows otherwise cost a second
  // cache line a run
  const int cs = c0 - (int)((reinterpret_cast<uintptr_t>(z + c0) & 15) / sizeof(T));
  // Elements at .. at + 7 of the row, -inf for those outside [c0, c1).
  auto load = [&](int at, float(&y)[8]) {
    if (at >= c0 && at + 8 <= c1) {
      load_run8(z + at, y);
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j) y[j] = -__builtin_inff();
      if (at + 8 > c0 && at < c1) {
#pragma unroll
        for (int j = 0; j < 8; ++j)
          if (at + j >= c0 && at + j < c1) y[j] = (float)z[at + j];
      }
    }
  };
  auto chunk = [&](auto whole, int c) {   // whole: every run of the chunk is
    constexpr bool kWhole = decltype(whole)::value;
    float x[U][8];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int at = c + 8 * (u * THR + t);
      if (kWhole)
        load_run8(z + at, x[u]);
      else
        load(at, x[u]);
    }
    float mxu[U], mx;
#pragma unroll
    for (int u = 0; u < U; ++u) {
      mxu[u] = x[u][0];
#pragma unroll
      for (int j = 1; j < 8; ++j) mxu[u] = fmaxf(mxu[u], x[u][j]);
      mx = u == 0 ? mxu[0] : fmaxf(mx, mxu[u]);
    }
    if (mx > st.m) lp_raise(st, mx);
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const float d = x[u][j] - st.m;
        const float e = fast_exp2(d * kLog2e);
        st.l += e;
        st.s += e * fmaxf(d, kFar);
      }
    if (TOP) {
      // the sums end here: left to itself the compiler carries their 32 terms past the bound, at 117 registers and
      // half the waves (69 registers with this line)
      asm volatile("" : "+v"(st.l), "+v"(st.s));
      ++done;
      if (done == next) {
        // The k-th largest of 64 maxima (256 for more than 24 alternatives), by the upper halves of
        // their keys: those of the waves' lanes together, lane by lane.  (A lane that holds NaN counts
        // with its largest other value: still one of its elements' keys or less.)
        const bool any = cs + 8 * t < c1;
        const uint32_t mine = any ? value_key(st.l == 0.0f ? -__builtin_inff() : st.m) >> 16 : 0u;
        uint32_t kth;
        if (W == 1) {
          const uint32_t v[1] = {mine};
          kth = lp_kth<1>(v, a.k);
        } else {
          // two buffers in turn: the next bound's maxima are not written over ones still being read
          keys_s[turn][t] = mine;
          __syncthreads();
          uint32_t v[4] = {0, 0, 0, 0};
#pragma unroll
          for (int i = 0; i < W; ++i) {
            const uint32_t o = keys_s[turn][64 * i + (t & 63)];
            v[i & 3] = o > v[i & 3] ? o : v[i & 3];
          }
          turn ^= 1;
          if (a.k > 24) {
            kth = lp_kth<4>(v, a.k);
          } else {
            uint32_t u[1] = {v[0]};
#pragma unroll
            for (int i = 1; i < 4; ++i) u[0] = v[i] > u[0] ? v[i] : u[0];
            kth = lp_kth<1>(u, a.k);
          }
        }
        thr = max(kth << 16, kMasked + 1);
        thr_z = key_value((uint64_t)thr << 32);
        next *= 4;
      }
      // the runs with an element at or above the bound: few, noted for the end
      uint32_t runs = 0;
#pragma unroll
      for (int u = 0; u < U; ++u) runs |= (mxu[u] < thr_z ? 0u : 1u) << u;
      if (st.l != st.l) runs = (1u << U) - 1;
      while (runs != 0) {
        const int i = atomicAdd(&nruns_s[sub], 1);
        if (i < RUNS) hist[sub][i] = (uint32_t)(c + 8 * ((__ffs(runs) - 1) * THR + t));
        runs &= runs - 1;
      }
    }
  };
  int c = cs;
  if (c < c0 && c < c1) {
    chunk(std::false_type{}, c);
    c += CH;
  }
  for (; c + CH <= c1; c += CH) chunk(std::true_type{}, c);
  if (c < c1) chunk(std::false_type{}, c);

  // the row's (or the part's) sums
  st = lp_group<W>(st, st_s);
  const bool split = ROWS == 1 && a.nsp > 1;
  float logl = 0.0f;
  if (live && t == 0 && split) a.part[row * a.nsp + part] = make_float4(st.m, st.l, st.s, 0.0f);
  if (live && !split) {
    if (t == 0) lp_finish(a, row, st, zt, has_t);
    logl = st.l == 0.0f ? -__builtin_inff() : logf(st.l);
  }

  if (TOP) {
    sync();
    const int nruns = nruns_s[sub], want_all = min(a.k, c1 - c0);
    if (nruns <= RUNS) {
      for (int i = t; i < nruns; i += THR) {
        const int at = (int)hist[sub][i];
        float y[8];
        load(at, y);
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          if (at + j >= c0 && at + j < c1 && value_key(y[j]) >= thr) {
            const int n = atomicAdd(&count_s[sub], 1);
            if (n < CAP) list[n] = elem_key(y[j], at + j);
          }
        }
      }
      sync();
    }
    int count = count_s[sub];
    if (nruns > RUNS || count > CAP || count < want_all) {
      // exact selection: the k-th key digit by digit from the top, then the keys at or above it
      const int lane = t & 63;
      uint64_t prefix = 0;
      uint32_t want = (uint32_t)want_all;
      sync();
      for (int sh = 56; sh >= 0; sh -= 8) {
        // digits that all keys of the prefix share: a short row's upper index bits, the lower half of a bf16 value's
        // key (ones below zero and for NaN)
        const bool low = sizeof(T) == 2 && (sh == 40 || sh == 32);
        if (low || (sh == 24 && a.V <= 1 << 24) || (sh == 16 && a.V <= 1 << 16)) {
          const bool ones = !low || prefix >> 63 == 0 || prefix >> 48 == 0xffff;
          prefix |= (uint64_t)(ones ? 255 : 0) << sh;
          continue;
        }
        for (int i = t; i < 256; i += THR) hist[sub][i] = 0;
        sync();
        for (int at = cs + 8 * t; at < c1; at += 8 * THR) {
          float y[8];
          load(at, y);
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            const uint64_t key = elem_key(y[j], at + j);
            const bool in = at + j >= c0 && at + j < c1 && (sh == 56 || (key >> (sh + 8)) == (prefix >> (sh + 8)));
            const uint32_t digit = (key >> sh) & 255;
            // ties are what comes here most: the lanes with the first one's digit are counted together
            if (in) {
              const uint32_t first = __builtin_amdgcn_readfirstlane(digit);
              const uint64_t same = __ballot(digit == first);
              if (digit != first)
                atomicAdd(&hist[sub][digit], 1u);
              else if (lane == __ffsll((unsigned long long)same) - 1)
                atomicAdd(&hist[sub][first], (uint32_t)__popcll(same));
            }
          }
        }
        sync();
        // the digit: every wave by itself, four digits a lane, the keys above a lane's by a scan
        uint32_t n[4], suf = 0;
#pragma unroll
        for (int i = 0; i < 4; ++i) suf += n[i] = hist[sub][4 * lane + i];
        const uint32_t own = suf;
#pragma unroll
        for (int o = 1; o < 64; o <<= 1) {
          const uint32_t v = __shfl_down(suf, o, kWave);
          suf += lane + o < 64 ? v : 0u;
        }
        uint32_t above = suf - own, d = 3, in = n[3];
        const uint64_t here = __ballot(above < want && suf >= want);
        for (int i = 2; i >= 0; --i)
          if (above + in < want) above += in, d = i, in = n[i];
        const int src = here == 0 ? 0 : __ffsll((unsigned long long)here) - 1;
        want -= __shfl(above, src, kWave);
        prefix |= (uint64_t)(4 * src + __shfl(d, src, kWave)) << sh;
        sync();
        if (__shfl(in, src, kWave) == want) break;   // every key of this prefix is one of the k best
      }
      if (t == 0) count_s[sub] = 0;
      sync();
      for (int at = cs + 8 * t; at < c1; at += 8 * THR) {
        float y[8];
        load(at, y);
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const uint64_t key = elem_key(y[j], at + j);
          if (at + j >= c0 && at + j < c1 && key >= prefix)
            list[atomicAdd(&count_s[sub], 1)] = key;   // k of them: the keys are all different
        }
      }
      sync();
      count = want_all;
    }
    if (live) {
      if (split) {
        uint64_t* out = a.part_top + (row * a.nsp + part) * a.k;
        for (int i = count + t; i < a.k; i += THR) out[i] = 0;
        lp_rank<THR>(list, count, a.k, t, [&](int r, uint64_t key) { out[r] = key; });
      } else {
        lp_rank<THR>(list, count, a.k, t, [&](int r, uint64_t key) {
          a.top_logp[row * a.k + r] = st.l == 0.0f ? -__builtin_inff() : (key_value(key) - st.m) - logl;
          a.top_idx[row * a.k + r] = (int64_t)(uint32_t)~(uint32_t)key;
        });
      }
    }
  }
}

// Larger of two keys over the wave, in every lane.
__device__ __forceinline__ uint64_t wave_max_key(uint64_t key) {
  const uint32_t hi = wave_reduce_u32<true>((uint32_t)(key >> 32));
  const uint32_t lo = wave_reduce_u32<true>((uint32_t)(key >> 32) == hi ? (uint32_t)key : 0u);
  return ((uint64_t)hi << 32) | lo;
}

// Joins the parts of a split row: one wave a row, one lane a part.  The parts'
// lists are sorted, so the k best come off their heads one after the other.
template <typename T>
__global__ __launch_bounds__(64) void k_logprob_join(const LpArgs a) {
  extern __shared__ uint64_t jlist[];
  const int64_t row = blockIdx.x;
  const int t = threadIdx.x;
  float zt = 0.0f;
  const bool has_t = t == 0 && lp_target<T>(a, row, zt);
  LpState st{kLowest, 0.0f, 0.0f};
  if (t < a.nsp) {
    const float4 p = a.part[row * a.nsp + t];
    st = LpState{p.x, p.y, p.z};
  }
  const int n = a.nsp * a.k;
  for (int i = t; i < n; i += 64) jlist[i] = a.part_top[row * n + i];
  float none[3][1];
  st = lp_group<1>(st, none);
  const float logl = st.l == 0.0f ? -__builtin_inff() : logf(st.l);
  if (t == 0) lp_finish(a, row, st, zt, has_t);
  __syncthreads();
  int at = t * a.k;
  const int end = t < a.nsp ? at + a.k : at;
  uint64_t head = at < end ? jlist[at] : 0, out = 0;
  for (int r = 0; r < a.k; ++r) {
    const uint64_t best = wave_max_key(head);
    if (t == r) out = best;
    if (head == best) {      // one lane: keys are all different (and k of them are no 0)
      ++at;
      head = at < end ? jlist[at] : 0;
    }
  }
  if (t < a.k) {
    a.top_logp[row * a.k + t] = st.l == 0.0f ? -__builtin_inff() : (key_value(out) - st.m) - logl;
    a.top_idx[row * a.k + t] = (int64_t)(uint32_t)~(uint32_t)out;
  }
}

struct LpBwdArgs {
  const void* z;
  const int64_t* target;        // or null
  const float2* stat;
  const float *entropy, *dlogp, *dent;   // dlogp, dent: or null
  void* dz;
  int64_t rows;
  int V, units;                 // units of a row
};

constexpr int kLpBwdRuns = 4;
constexpr int kLpBwdUnit = 64 * 8 * kLpBwdRuns;   // elements a wave takes

template <typename T, bool ENT>
__global__ __launch_bounds__(256) void k_logprob_bwd(const LpBwdArgs a) {
  const int64_t unit = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
  const int64_t row = unit / a.units;
  if (row >= a.rows) return;
  const int lane = threadIdx.x & 63;
  const int c = (int)(unit % a.units) * kLpBwdUnit + 8 * lane;
  const T* z = static_cast<const T*>(a.z) + row * a.V;
  T* dz = static_cast<T*>(a.dz) + row * a.V;
  int64_t tg = a.target == nullptr ? -1 : a.target[row];
  const float2 st = a.stat[row];
  const bool empty = st.y == -__builtin_inff();   // nothing in the row: no gradient
  const float dl = a.dlogp == nullptr || tg < 0 || tg >= a.V || empty ? 0.0f : a.dlogp[row];
  if (dl == 0.0f) tg = -1;
  const float dh = ENT && !empty ? a.dent[row] : 0.0f;
  const bool zero = dl == 0.0f && dh == 0.0f;
  const float log2l = st.y * kLog2e;
  const float hh = ENT ? a.entropy[row] - st.y : 0.0f;
  float x[kLpBwdRuns][8];
  if (!zero) {
#pragma unroll
    for (int u = 0; u < kLpBwdRuns; ++u) {
      const int at = c + 512 * u;
      load_run8(z + at, a.V - at, x[u]);
    }
  }
#pragma unroll
  for (int u = 0; u < kLpBwdRuns; ++u) {
    const int at = c + 512 * u;
    if (at >= a.V) break;
    float d[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      if (zero) {
        d[j] = 0.0f;
      } else {
        const float y = x[u][j] - st.x;
        const float p = fast_exp2(y * kLog2e - log2l);
        d[j] = ENT ? -p * (dl + dh * (fmaxf(y, kFar) + hh)) : -p * dl;
      }
      if (tg == at + j) d[j] += dl;
    }
    store_run8(dz + at, a.V - at, d);
  }
}

// Waves of a row: one up to 2048 elements, and up to 8192 where the rows give
// every compute unit sixteen waves by themselves: no barriers, and no idle lanes
// where a row is little more than a workgroup's chunk (32768 x 2500 in bf16 with
// one wave 48 to 53 us, with four 82; 8192 x 8192 with 5 alternatives 33 and 39,
// without them 30 and 29; more than 24 alternatives overfill one wave's list:
// 97 us with 40, and 49 with four waves; longer rows gain a tenth, at four times the additions in a lane).  Sixteen where the rows leave most of
// the chip's waves idle (a row of 32000 in 16 bits is then one chunk); else four.
// A row of more than 256 KiB is split where there are not enough of them
// either, into parts of 8192 elements or more, two for every compute unit: one
// workgroup's loads would take longer than the second launch.
static int lp_waves(int64_t rows, int V, int k, int cu) {
  if (V <= 2048 || (V <= 8192 && k <= 24 && rows >= 16 * cu)) return 1;
  return rows <= 2 * cu ? 16 : 4;
}
static int lp_parts(int64_t rows, int V, int esize, int cu) {
  if ((int64_t)V * esize <= 256 * 1024 || rows >= 2 * cu) return 1;
  int64_t want = (2LL * cu + rows - 1) / rows;
  const int chunks = (V + 8191) / 8192;
  if (want > chunks) want = chunks;
  if (want > 64) want = 64;   // a lane each in the join
  const int per = (int)((chunks + want - 1) / want);
  return (chunks + per - 1) / per;
}
static int lp_seg(int V, int nsp) {
  if (nsp <= 1) return V;
  const int chunks = (V + 8191) / 8192;
  return ((chunks + nsp - 1) / nsp) * 8192;
}

template <typename T, bool TOP>
static int logprob_launch(LpArgs a, hipStream_t s) {
  const int w = a.nsp > 1 ? 4 : lp_waves(a.rows, a.V, a.k, device_cu_count(s));
  if (w == 1) {
    // as many runs in flight as the row has: 32768 x 512 takes 13 us with one run, 22 with four
    const unsigned grid = (unsigned)((a.rows + 3) / 4);
    if (a.V <= 512)
      k_logprob<T, 1, 1, TOP><<<grid, 256, 0, s>>>(a);
    else if (a.V <= 1024)
      k_logprob<T, 1, 2, TOP><<<grid, 256, 0, s>>>(a);
    else
      k_logprob<T, 1, 4, TOP><<<grid, 256, 0, s>>>(a);
  } else if (w == 4) {
    // runs in flight against waves: 2047 x 50257 with 5 alternatives takes 56 us at four runs, 52 at three, 50 at two
    k_logprob<T, 4, 2, TOP><<<(unsigned)(a.rows * a.nsp), 256, 0, s>>>(a);
  } else {
    // 256 x 131072 without alternatives: 13.5 us at two runs, 15.5 at four; 32 x 32000 with 20: 8.8 and 8.5
    k_logprob<T, 16, TOP ? 4 : 2, TOP><<<(unsigned)a.rows, 1024, 0, s>>>(a);
  }
  if (a.nsp > 1) k_logprob_join<T><<<(unsigned)a.rows, 64, (size_t)a.nsp * a.k * 8, s>>>(a);
  return nsa_launch_status();
}

}  // namespace nsa

static bool lp_shape_ok(int64_t rows, int V, int k) {
  return rows >= 0 && rows <= (1LL << 25) && V >= 1 && V <= (1 << 28) && k >= 0 && k <= nsa::kLpTopMax && k <= V;
}

extern "C" size_t nsa_logprob_workspace(int64_t rows, int V, int k, void* stream) {
  using namespace nsa;
  if (!lp_shape_ok(rows, V, k)) return 0;
  if (rows == 0) return 16;
  const int nsp = lp_parts(rows, V, 4, device_cu_count(static_cast<hipStream_t>(stream)));   // (float32: no fewer)
  return nsp <= 1 ? 16 : (size_t)rows * nsp * (16 + 8 * (size_t)k);
}

extern "C" int nsa_logprob_fwd(const void* z, const int64_t* target, float* logp, float* entropy, float* stat,
                               float* top_logp, int64_t* top_idx, void* workspace, size_t workspace_bytes,
                               int64_t rows, int V, int k, int dtype, void* stream) {
  using namespace nsa;
  NSA_CHECK(lp_shape_ok(rows, V, k), NSA_ERR_SHAPE);
  NSA_CHECK(dtype == NSA_F32 || dtype == NSA_BF16, NSA_ERR_DTYPE);
  if (rows == 0) return NSA_OK;
  NSA_CHECK(z != nullptr && (logp == nullptr || target != nullptr), NSA_ERR_ARG);
  NSA_CHECK(k == 0 || (top_logp != nullptr && top_idx != nullptr), NSA_ERR_ARG);
  const hipStream_t s = static_cast<hipStream_t>(stream);
  const int nsp = lp_parts(rows, V, dtype == NSA_BF16 ? 2 : 4, device_cu_count(s));
  LpArgs a{z, target, logp, entropy, reinterpret_cast<float2*>(stat), top_logp, top_idx, nullptr, nullptr, rows, V,
           k, nsp, lp_seg(V, nsp)};
  if (nsp > 1) {
    NSA_CHECK(workspace != nullptr && workspace_bytes >= (size_t)rows * nsp * (16 + 8 * (size_t)k), NSA_ERR_WORKSPACE);
    a.part = static_cast<float4*>(workspace);
    a.part_top = reinterpret_cast<uint64_t*>(static_cast<char*>(workspace) + (size_t)rows * nsp * 16);
  }
  // 2^21 rows a launch: a grid holds less than 2^32 threads (rows that are split are far fewer)
  for (int64_t r0 = 0; r0 < rows; r0 += kLpSlice) {
    LpArgs b = a;
    b.rows = rows - r0 < kLpSlice ? rows - r0 : kLpSlice;
    b.z = static_cast<const char*>(z) + r0 * V * (dtype == NSA_BF16 ? 2 : 4);
    if (target != nullptr) b.target = target + r0;
    if (logp != nullptr) b.logp = logp + r0;
    if (entropy != nullptr) b.entropy = entropy + r0;
    if (stat != nullptr) b.stat = a.stat + r0;
    if (k > 0) {
      b.top_logp = top_logp + r0 * k;
      b.top_idx = top_idx + r0 * k;
    }
    int rc;
    if (dtype == NSA_BF16)
      rc = k > 0 ? logprob_launch<bf16, true>(b, s) : logprob_launch<bf16, false>(b, s);
    else
      rc = k > 0 ? logprob_launch<float, true>(b, s) : logprob_launch<float, false>(b, s);
    if (rc != NSA_OK) return rc;
  }
  return NSA_OK;
}

extern "C" int nsa_logprob_bwd(const void* z, const int64_t* target, const float* stat, const float* entropy,
                               const float* dlogp, const float* dent, void* dz, int64_t rows, int V, int dtype,
                               void* stream) {
  using namespace nsa;
  NSA_CHECK(lp_shape_ok(rows, V, 0), NSA_ERR_SHAPE);
  NSA_CHECK(dtype == NSA_F32 || dtype == NSA_BF16, NSA_ERR_DTYPE);
  if (rows == 0) return NSA_OK;
  NSA_CHECK(z != nullptr && stat != nullptr && dz != nullptr && (dent == nullptr || entropy != nullptr), NSA_ERR_ARG);
  const hipStream_t s = static_cast<hipStream_t>(stream);
  const int units = (V + kLpBwdUnit - 1) / kLpBwdUnit;
  const int64_t slice = (1LL << 25) / units > 1 ? (1LL << 25) / units : 1;   // rows of one launch: 2^31 threads
  const size_t es = dtype == NSA_BF16 ? 2 : 4;
  for (int64_t r0 = 0; r0 < rows; r0 += slice) {
    const int64_t n = rows - r0 < slice ? rows - r0 : slice;
    const unsigned grid = (unsigned)((n * units + 3) / 4);
    const LpBwdArgs a{static_cast<const char*>(z) + r0 * V * es,
                      target == nullptr ? nullptr : target + r0,
                      reinterpret_cast<const float2*>(stat) + r0,
                      entropy == nullptr ? nullptr : entropy + r0,
                      dlogp == nullptr ? nullptr : dlogp + r0,
                      dent == nullptr ? nullptr : dent + r0,
                      static_cast<char*>(dz) + r0 * V * es,
                      n, V, units};
    if (dtype == NSA_BF16) {
      if (dent != nullptr)
        k_logprob_bwd<bf16, true><<<grid, 256, 0, s>>>(a);
      else
        k_logprob_bwd<bf16, false><<<grid, 256, 0, s>>>(a);
    } else {
      if (dent != nullptr)
        k_logprob_bwd<float, true><<<grid, 256, 0, s>>>(a);
      else
        k_logprob_bwd<float, false><<<grid, 256, 0, s>>>(a);
    }
    const int rc = nsa_launch_status();
    if (rc != NSA_OK) return rc;
  }
  return NSA_OK;
}
