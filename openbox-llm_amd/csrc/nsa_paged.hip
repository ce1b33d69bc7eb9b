// Attention of one new token of every sequence over a paged key-value cache,
// with the append of its key and value rows, and the writing of whole prompts.
//
//   pages  [n_pages][Hkv][P][D]  keys and values; P a multiple of 16
//   table  [B][max_pages]        position p of sequence b lies in page table[b][p / P], row p % P
//   lens   [B]                   keys of each sequence before the step
//   out[b][h] = softmax(scale q K^T) V over the keys 0 .. n-1 of KV head h / (Hq / Hkv)
//
// A step is bound by reading each key and value row once.  The keys of all
// sequences and KV heads (and head tiles of up to 32 query heads) are one list
// of units of 128 keys, cut into equal shares, one to a workgroup: sequences of
// unlike lengths then end together.  A share is a few pieces, each of one
// sequence and head; within a piece each of the four waves takes tiles of 32
// keys in turn, with the running maximum and sum of the softmax, and the four
// are joined in LDS.  A sequence and head whose keys are one piece is written
// out at once; else the pieces' unnormalised outputs go to the workspace and a
// second launch joins them.
//
// Rows go from memory to the matrix operands without LDS.  K: lane (g, c) of
// S^T = K Q^T holds 8 d of key c, so 16 bytes of the row.  V: O^T = V^T P^T wants 8
// keys of one d a lane.  Lane (g, c) loads D / 16 consecutive d (c's) of each of
// its 8 keys (8 g ..): every load instruction reads whole rows, and the operand
// of tile i, whose row c stands for d = c D / 16 + i, is element i of the 8
// loads -- a transpose inside the lane.  P is split in two bf16 parts (high
// and rest) that go through the products one after the other: the
// matrix unit has time to spare here, and the output then carries no
// rounding but its own.
//
// A page's address is formed in 64 bits, for runs of 16 keys (a run lies in one
// page).  Runs whose table entry is outside 0 .. n_pages-1 hold no keys.
// Rows at and past a sequence's length may hold anything: their scores are
// replaced and their values zeroed before they meet a weight.  The step's own
// row is taken from the caller's new rows, not from the page it is written to,
// so that no read waits for that write.
//
// Measured (MI355X, bf16, 64:4 heads of 128 unless said): 32 sequences of 4K to
// 32K 214 us, 5.6 TB/s of keys and values, bound by memory; one of 32K 19.4 us
// (12.3 at the rate of a large copy), of which the join is 4 and the chain
// length - table - rows before the first score about 3; 200 chats of up to 900
// (12:2 heads of 64) 15.7 us, bound by the tiles of the longest.  More than 32
// heads a KV head are tiles that each read the keys and values again: 64 of up to 2K
// take 19 us at 16:1, 26 at 32:1, 29 at 40:1.  Prompts go into pages at the rate of a
// copy (32K of 4 heads of 128 23.5 us, 5.7 TB/s).
#include "nsa_launch.h"
#include "nsa_paged_index.h"
#include "nsa_tiles.h"

namespace nsa {

constexpr int kUnit = 128;   // keys of a unit: a tile for each wave
// The running maximum's start, and the score of a key that is not there: at or below every finite score (a sentinel
// within their range would take weight from rows whose scores are all below it).
constexpr float kLowScore = -3.402823466e38f;

struct PagedArgs {
  const void *q, *k_new, *v_new;     // [B][Hq][D], [B][Hkv][D] (null: no append)
  void *kp, *vp;
  const int32_t *table, *lens;
  int32_t* lens_out;                 // or null
  void* out;
  float* lse;                        // or null
  float* part_o;                     // [W + R][16 NT][D]: piece of share w and row r at w + r
  float2* part_ml;                   // [W + R][16 NT]
  int2* row_info;                    // [R] first and last share of a row in pieces, (-1, -1) of one piece
  int B, Hq, Hkv, G, HT, P, rpp;     // HT: head tiles of a KV head; rpp: runs of 16 in a page
  int max_pages, n_pages, W;         // W: shares of the list, or 0: a workgroup a row
  int limit;                         // no row is appended at or past it (at most max_pages * P)
  float sl2;                         // scale * log2 e
};

// Keys that sequence b attends, twice, plus 1 where the last of them is the row it would append.  (Where
// that row has no page, its run has none either: it is neither attended nor written.  Past the limit there is
// no such row, page or not.)
__device__ __forceinline__ uint32_t paged_keys(const PagedArgs& a, int b) {
  const int cap = a.max_pages * a.P;
  const int len = a.lens[b];
  if (a.k_new != nullptr && len >= 0 && len < a.limit) return 2u * ((uint32_t)len + 1u) + 1u;
  return 2u * (uint32_t)(len < 0 ? 0 : (len < cap ? len : cap));
}
// Units of a row of n keys: one at least, so that an empty row is written too.
__device__ __forceinline__ int paged_units(uint32_t keys) {
  const int n = (int)(keys >> 1);
  return n <= kUnit ? 1 : (n + kUnit - 1) / kUnit;
}

__device__ __forceinline__ float paged_lse(float m, float l) {
  return l > 0.0f ? (m + __log2f(l)) * kLn2 : (l == 0.0f ? kLseEmpty : l);   // (NaN stays)
}

__device__ __forceinline__ int64_t run_base(const PagedArgs& a, int b, int hkv, int run, int D) {
  return paged_run(a.table + (int64_t)b * a.max_pages, run, a.rpp, a.max_pages, a.n_pages, a.Hkv, hkv, D);
}

// VL = D / 16 consecutive elements of a row
template <typename T, int VL> struct VRun {
  T v[VL];
};
template <> struct VRun<bf16, 8> { bf16x8 v; };
template <> struct VRun<bf16, 4> { bf16x4 v; };
template <> struct VRun<float, 8> { f32x4 v4[2]; };
template <> struct VRun<float, 4> { f32x4 v4[1]; };
template <typename T, int VL> __device__ __forceinline__ T vrun_elem(const VRun<T, VL>& r, int i) {
  if constexpr (sizeof(T) == 4 && VL >= 4)
    return r.v4[i >> 2][i & 3];
  else
    return r.v[i];
}
template <typename T, int VL> __device__ __forceinline__ VRun<T, VL> vrun_load(const T* p) {
  VRun<T, VL> r;
  if constexpr (sizeof(T) == 2 && VL == 8)
    r.v = *reinterpret_cast<const bf16x8*>(p);
  else if constexpr (sizeof(T) == 2 && VL == 4)
    r.v = *reinterpret_cast<const bf16x4*>(p);
  else if constexpr (sizeof(T) == 4 && VL >= 4) {
#pragma unroll
    for (int i = 0; i < VL / 4; ++i) r.v4[i] = *reinterpret_cast<const f32x4*>(p + 4 * i);
  } else {
#pragma unroll
    for (int i = 0; i < VL; ++i) r.v[i] = p[i];
  }
  return r;
}
template <typename T, int VL> __device__ __forceinline__ VRun<T, VL> vrun_zero() {
  VRun<T, VL> r;
  __builtin_memset(&r, 0, sizeof(r));
  return r;
}

// NT: tiles of 16 query heads.
template <typename T, int D, int NT>
__global__ __launch_bounds__(256, 2) void k_paged(const PagedArgs a) {
  constexpr int KC = Dims<D>::KC, DT = Dims<D>::DT, VL = D / 16;
  constexpr bool SPLIT_P = sizeof(T) == 2;
  constexpr int QF = sizeof(Frag<T>) / 16;           // 16-byte pieces of an operand
  __shared__ f32x4 qs[NT][KC][QF][64];                // the queries as operands, one piece a lane
  __shared__ float so[4][16][D + 4];                  // the waves' outputs
  __shared__ float sm[4][16], sl[4][16];
  __shared__ __align__(16) T rows_new[2][D];          // the appended row
  __shared__ int wsum[4], found[2];
  __shared__ uint32_t seq_keys[256];                  // of every sequence, where there are no more than 256
  const int lane = threadIdx.x & 63, g = lane >> 4, c = lane & 15;
  const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int M = a.Hkv * a.HT;                         // rows of a sequence
  const T* kp = static_cast<const T*>(a.kp);
  const T* vp = static_cast<const T*>(a.vp);

  // This workgroup's units: [x, x1) of the list, the first of them in row m of
  // sequence b, whose `units` units start at row0.
  int x, x1, row0, W = 0, share = 0, more = 0;        // W shares: `more` of share + 1 units, then of share
  int b, m, units;
  uint32_t keys;
  if (a.W == 0) {                                     // a row each: the list is that row
    b = (int)(blockIdx.x / (unsigned)M);
    m = (int)(blockIdx.x % (unsigned)M);
    keys = paged_keys(a, b);
    units = paged_units(keys);
    x = row0 = 0;
    x1 = units;
  } else {
    // Each thread counts the units of its sequences; the one whose range holds x finds the sequence.
    const int per = (a.B + 255) / 256;
    const int b_lo = min(a.B, (int)threadIdx.x * per), b_hi = min(a.B, b_lo + per);
    int mine = 0;
    for (int i = b_lo; i < b_hi; ++i) {
      keys = paged_keys(a, i);
      mine += paged_units(keys);
    }
    if (per == 1 && b_lo < b_hi) seq_keys[b_lo] = keys;
    int incl = mine;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
      const int v = __shfl_up(incl, o, 64);
      if (lane >= o) incl += v;
    }
    if (lane == 63) wsum[w] = incl;
    __syncthreads();
    int before = incl - mine, U = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if (i < w) before += wsum[i];
      U += wsum[i];
    }
    U *= M;
    before *= M;
    W = U < a.W ? U : a.W;                            // shares of one unit at least: a row's pieces have no gaps
    if ((int)blockIdx.x >= W) return;                 // (uniform)
    share = U / W;
    more = U - share * W;
    x = (int)blockIdx.x * share + min((int)blockIdx.x, more);
    x1 = x + share + ((int)blockIdx.x < more ? 1 : 0);
    if (x >= before && x < before + mine * M) {
      int i = b_lo;
      if (per > 1) {
        for (;; ++i) {
          const int u = paged_units(paged_keys(a, i)) * M;
          if (x < before + u) break;
          before += u;
        }
      }
      found[0] = i;
      found[1] = before;
    }
    __syncthreads();
    b = __builtin_amdgcn_readfirstlane(found[0]);
    keys = a.B <= 256 ? (uint32_t)__builtin_amdgcn_readfirstlane((int)seq_keys[b]) : paged_keys(a, b);
    units = paged_units(keys);
    m = (x - found[1]) / units;
    row0 = found[1] + m * units;
  }

  while (x < x1) {
    const int hkv = m / a.HT, ht = m - hkv * a.HT;
    const int t0 = x - row0;
    const int t1 = x1 - row0 < units ? x1 - row0 : units;
    const bool one = t0 == 0 && t1 == units;          // the row in one piece
    const int n = (int)(keys >> 1), pos = (keys & 1u) ? n - 1 : -1;
    const int c0 = kUnit * t0, c1 = min(n, kUnit * t1);
    const int row = b * M + m;
    const T* kn = static_cast<const T*>(a.k_new) + ((int64_t)b * a.Hkv + hkv) * D;
    const T* vn = static_cast<const T*>(a.v_new) + ((int64_t)b * a.Hkv + hkv) * D;

    // this wave's tiles: 32 keys every 128; lane i looks up run i of the current 32 tiles
    const int my0 = c0 + 32 * w;
    const int ntile = c1 > my0 ? (c1 - my0 + kUnit - 1) / kUnit : 0;
    int64_t base = -1;
    auto look_up = [&](int i) {   // runs of tiles i .. i + 31
      const int tile = i + (lane >> 1), key = my0 + kUnit * tile + 16 * (lane & 1);
      base = tile < ntile && key < c1 ? run_base(a, b, hkv, key >> 4, D) : -1;
    };
    auto run_at = [&](int i) -> int64_t {   // (i uniform, of the current 32 tiles)
      const uint32_t lo = (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)base, i & 63);
      const uint32_t hi = (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)((uint64_t)base >> 32), i & 63);
      return (int64_t)(((uint64_t)hi << 32) | lo);
    };
    // Loads of a tile: always the same number, whatever the tile holds, so that waiting for the keys does not
    // wait for what was asked for behind them.  Runs without a page read page 0 instead, and rows past the
    // length their own page's; the masks and fix_v() take out what is not there.
    Frag<T> kf[2][KC];       // keys kb + 8 (c >> 2) + 4 mt + (c & 3)
    VRun<T, VL> vr[8];       // keys kb + 8 g + j
    uint32_t vm;             // which of keys kb + 8 g .. + 7 are visible
    auto load_k = [&](int i) {
      if ((i & 31) == 0) look_up(i);
      const int64_t b0 = run_at(2 * i), b1 = run_at(2 * i + 1);
      vm = (g >= 2 ? b1 : b0) >= 0 ? range_mask(my0 + kUnit * i + 8 * g, 0, c1 - 1) : 0u;
      const int64_t base_k = c >= 8 ? b1 : b0;
      const T* at = kp + (base_k >= 0 ? base_k : 0) + (((8 * (c >> 2)) & 15) + (c & 3)) * D + 8 * g;
#pragma unroll
      for (int mt = 0; mt < 2; ++mt)
#pragma unroll
        for (int kc = 0; kc < KC; ++kc) {
          if (32 * kc + 8 * g < D)
            kf[mt][kc].load(at + 4 * mt * D + 32 * kc);
          else
            kf[mt][kc].zero();
        }
    };
    auto load_v = [&](int i) {   // (behind load_k of the same tile)
      const int64_t base_v = g >= 2 ? run_at(2 * i + 1) : run_at(2 * i);
      const T* at = vp + (base_v >= 0 ? base_v : 0) + ((8 * g) & 15) * D + VL * c;
#pragma unroll
      for (int j = 0; j < 8; ++j) vr[j] = vrun_load<T, VL>(at + j * D);
    };
    // The appended row in place of its page's, which another workgroup may be writing.
    auto new_k = [&](int i) {
#pragma unroll
      for (int mt = 0; mt < 2; ++mt) {
        if (my0 + kUnit * i + 8 * (c >> 2) + 4 * mt + (c & 3) == pos) {
#pragma unroll
          for (int kc = 0; kc < KC; ++kc)
            if (32 * kc + 8 * g < D) kf[mt][kc].load(&rows_new[0][32 * kc + 8 * g]);
        }
      }
    };
    // The values of keys that are not visible to 0 (a weight of 0 does not take NaN out), and the appended row.
    auto fix_v = [&](int i, uint32_t seen) {
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        if (my0 + kUnit * i + 8 * g + j == pos)
          vr[j] = vrun_load<T, VL>(&rows_new[1][VL * c]);
        if (((seen >> j) & 1u) == 0u) vr[j] = vrun_zero<T, VL>();
      }
    };
    // queries to LDS as operands: wave w takes every fourth.  They are asked for first: loads return in order.
    Frag<T> qf[(NT * KC + 3) / 4];
#pragma unroll
    for (int f = 0; f < NT * KC; f += 4) {
      const int nt = (f + w) / KC, kc = (f + w) % KC, hg = ht * 16 * NT + 16 * nt + c;
      if (f + w < NT * KC && hg < a.G && 32 * kc + 8 * g < D)
        qf[f / 4].load(static_cast<const T*>(a.q) + ((int64_t)b * a.Hq + (int64_t)hkv * a.G + hg) * D + 32 * kc + 8 * g);
      else
        qf[f / 4].zero();
    }
    if (ntile > 0) {
      load_k(0);
      load_v(0);
    }
#pragma unroll
    for (int f = 0; f < NT * KC; f += 4) {
      if (f + w < NT * KC) {
#pragma unroll
        for (int i = 0; i < QF; ++i)
          qs[(f + w) / KC][(f + w) % KC][i][lane] = reinterpret_cast<const f32x4*>(&qf[f / 4])[i];
      }
    }

    if (t0 == 0 && threadIdx.x == 0) {
      if (a.row_info != nullptr) {
        const int last = row0 + units - 1, big = more * (share + 1);   // the share of the row's last unit
        const int wl = last < big ? last / (share + 1) : more + (last - big) / share;
        a.row_info[row] = one ? make_int2(-1, -1) : make_int2((int)blockIdx.x, wl);
      }
      if (a.lens_out != nullptr && m == 0) {
        const int len = a.lens[b];
        const bool fits = len < a.limit &&
                          paged_new_pos(a.table + (int64_t)b * a.max_pages, len, a.P, a.max_pages, a.n_pages) >= 0;
        a.lens_out[b] = fits ? len + 1 : len;
      }
    }
    // the appended row: to LDS for this piece's tiles, and by the first head tile to its page
    if (pos >= c0 && pos < c1 && threadIdx.x < D) {
      const int d = threadIdx.x;
      const T k1 = kn[d], v1 = vn[d];
      rows_new[0][d] = k1;
      rows_new[1][d] = v1;
      const int64_t at = run_base(a, b, hkv, pos >> 4, D);
      if (ht == 0 && at >= 0) {
        static_cast<T*>(a.kp)[at + (int64_t)(pos & 15) * D + d] = k1;
        static_cast<T*>(a.vp)[at + (int64_t)(pos & 15) * D + d] = v1;
      }
    }
    __syncthreads();

    FwdAcc<D> acc[NT];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      acc[nt].init();
      acc[nt].m = kLowScore;
    }
    for (int i = 0; i < ntile; ++i) {
      // The next tile's keys are asked for as soon as this one's are used, its values likewise: a wave has one or
      // the other in flight at all times, in the registers of one tile.  (Two tiles ahead measured slower: 232
      // against 220 us for 32 sequences of up to 32K.)
      const int kb = my0 + kUnit * i;
      const bool has_new = pos >= kb && pos < kb + 32;
      if (has_new) new_k(i);
      f32x4 s[NT][2];
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        s[nt][0] = zero4();
        s[nt][1] = zero4();
#pragma unroll
        for (int kc = 0; kc < KC; ++kc) {
          Frag<T> q;
#pragma unroll
          for (int y = 0; y < QF; ++y) reinterpret_cast<f32x4*>(&q)[y] = qs[nt][kc][y][lane];
          mma(s[nt][0], kf[0][kc], q);
          mma(s[nt][1], kf[1][kc], q);
        }
      }
      const uint32_t seen = vm;
      const bool all = __all(seen == 0xffu);
      if (i + 1 < ntile) load_k(i + 1);
      Frag<T> ph[NT], pl[NT];
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        FwdAcc<D>& A = acc[nt];
        float sv[8], mx = kLowScore;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          sv[j] = ((seen >> j) & 1u) ? s[nt][j >> 2][j & 3] * a.sl2 : kLowScore;
          mx = fmaxf(mx, sv[j]);
        }
        mx = group4_max(mx);
        if (__any(mx > A.m)) {
          const float mn = fmaxf(A.m, mx);
          const float alpha = fast_exp2(A.m - mn);
          A.l *= alpha;
          A.m = mn;
#pragma unroll
          for (int dt = 0; dt < DT; ++dt) A.o[dt] *= alpha;
        }
        float p[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          p[j] = ((seen >> j) & 1u) ? fast_exp2(sv[j] - A.m) : 0.0f;
          A.l += p[j];
        }
        ph[nt].set(p);
        if constexpr (SPLIT_P) {
#pragma unroll
          for (int j = 0; j < 8; ++j) p[j] -= (float)ph[nt].elem(j);
          pl[nt].set(p);
        }
      }
      if (has_new || !all) fix_v(i, seen);
#pragma unroll
      for (int dt = 0; dt < DT; ++dt) {
        Frag<T> vf;
        if constexpr (sizeof(T) == 2) {
#pragma unroll
          for (int j = 0; j < 8; ++j) vf.v[j] = vrun_elem<T, VL>(vr[j], dt);
        } else {
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            vf.lo[j] = vrun_elem<T, VL>(vr[j], dt);
            vf.hi[j] = vrun_elem<T, VL>(vr[4 + j], dt);
          }
        }
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
          mma(acc[nt].o[dt], vf, ph[nt]);
          if constexpr (SPLIT_P) mma(acc[nt].o[dt], vf, pl[nt]);
        }
      }
      if (i + 1 < ntile) load_v(i + 1);
    }

    // join the four waves: their outputs against the common maximum, added in wave order
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      FwdAcc<D>& A = acc[nt];
      A.l = group4_sum(A.l);
      if (nt > 0) __syncthreads();
      if (g == 0) sm[w][c] = A.m, sl[w][c] = A.l;
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        float* p = &so[w][c][VL * (4 * g + r)];
#pragma unroll
        for (int dt = 0; dt < DT; ++dt) p[dt] = A.o[dt][r];
      }
      __syncthreads();
      // 16 threads a head
      const int hr = threadIdx.x >> 4, y = threadIdx.x & 15;
      const int hg = ht * 16 * NT + 16 * nt + hr;
      if (hg < a.G) {
        const float mj = fmaxf(fmaxf(sm[0][hr], sm[1][hr]), fmaxf(sm[2][hr], sm[3][hr]));
        float f[4], l = 0.0f;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          f[i] = fast_exp2(sm[i][hr] - mj);
          l += sl[i][hr] * f[i];
        }
        const float inv = !one ? 1.0f : (l > 0.0f ? 1.0f / l : 0.0f);
        float o[VL];
#pragma unroll
        for (int e = 0; e < VL; ++e) {
          const int d = VL * y + e;
          o[e] = (((so[0][hr][d] * f[0] + so[1][hr][d] * f[1]) + so[2][hr][d] * f[2]) + so[3][hr][d] * f[3]) * inv;
        }
        if (!one) {
          const int64_t slot = ((int64_t)blockIdx.x + row) * (16 * NT) + 16 * nt + hr;
          float* out = a.part_o + slot * D + VL * y;
#pragma unroll
          for (int e = 0; e < VL; ++e) out[e] = o[e];
          if (y == 0) a.part_ml[slot] = make_float2(mj, l);
        } else {
          const int64_t head = (int64_t)b * a.Hq + (int64_t)hkv * a.G + hg;
          T* out = static_cast<T*>(a.out) + head * D + VL * y;
#pragma unroll
          for (int e = 0; e < VL; ++e) out[e] = (T)o[e];
          if (a.lse != nullptr && y == 0) a.lse[head] = paged_lse(mj, l);
        }
      }
    }

    x += t1 - t0;
    if (x < x1) {                                     // on to the next row
      row0 += units;
      if (++m == M) {
        m = 0;
        ++b;
        keys = a.B <= 256 ? (uint32_t)__builtin_amdgcn_readfirstlane((int)seq_keys[b]) : paged_keys(a, b);
        units = paged_units(keys);
      }
    }
  }
}

// Joins the pieces of a head: one workgroup of W waves, which take pieces in
// turn.  Heads written in one piece are left as they are.
template <typename T, int D, int W>
__global__ __launch_bounds__(64 * W) void k_paged_join(const PagedArgs a, int NT) {
  __shared__ float so[W][D], sm[W], sl[W];
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
  const int64_t head = blockIdx.x;
  const int b = (int)(head / a.Hq), h = (int)(head % a.Hq);
  const int hkv = h / a.G, hg = h % a.G, ht = hg / (16 * NT);
  const int row = (b * a.Hkv + hkv) * a.HT + ht;
  const int2 ri = a.row_info[row];
  if (ri.x < 0) return;                               // (uniform)
  const int np = ri.y - ri.x + 1;
  const int64_t slot0 = ((int64_t)ri.x + row) * (16 * NT) + (hg - ht * 16 * NT);
  const float2* ml = a.part_ml + slot0;
  const float* po = a.part_o + slot0 * D;
  const int step = 16 * NT;                           // slots from a piece to the next
  // Pieces w, w + W, ... eight at a time, all asked for at once; a running maximum, the waves' own joined below.
  constexpr int E = D >= 64 ? D / 64 : 1;
  float m = kLowScore, l = 0.0f, o[E];
#pragma unroll
  for (int e = 0; e < E; ++e) o[e] = 0.0f;
  for (int i0 = w; i0 < np; i0 += 8 * W) {
    float2 s[8];
    float v[8][E], mx = m;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const int i = i0 + j * W;
      s[j] = i < np ? ml[(int64_t)i * step] : make_float2(kLowScore, 0.0f);
#pragma unroll
      for (int e = 0; e < E; ++e)
        v[j][e] = i < np && E * lane + e < D ? po[(int64_t)i * step * D + E * lane + e] : 0.0f;
    }
#pragma unroll
    for (int j = 0; j < 8; ++j) mx = fmaxf(mx, s[j].x);
    const float f0 = fast_exp2(m - mx);
    l *= f0;
#pragma unroll
    for (int e = 0; e < E; ++e) o[e] *= f0;
    m = mx;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const float f = fast_exp2(s[j].x - m);
      l += s[j].y * f;
#pragma unroll
      for (int e = 0; e < E; ++e) o[e] += v[j][e] * f;
    }
  }
#pragma unroll
  for (int e = 0; e < E; ++e)
    if (E * lane + e < D) so[w][E * lane + e] = o[e];
  if (lane == 0) sm[w] = m, sl[w] = l;
  __syncthreads();
  m = sm[0];
#pragma unroll
  for (int i = 1; i < W; ++i) m = fmaxf(m, sm[i]);
  l = 0.0f;
#pragma unroll
  for (int i = 0; i < W; ++i) l += sl[i] * fast_exp2(sm[i] - m);
  const float inv = l > 0.0f ? 1.0f / l : 0.0f;
  if ((int)threadIdx.x < D) {
    const int d = threadIdx.x;
    float v = 0.0f;
#pragma unroll
    for (int i = 0; i < W; ++i) v += so[i][d] * fast_exp2(sm[i] - m);
    static_cast<T*>(a.out)[head * D + d] = (T)(v * inv);
  }
  if (a.lse != nullptr && threadIdx.x == 0) a.lse[head] = paged_lse(m, l);
}

// Rows [B][Hkv][Tn][D] to positions lens[b] .. lens[b] + count[b] - 1: all of a
// sequence's rows, or none where they do not all have a page.
template <typename T>
__global__ __launch_bounds__(256) void k_paged_append(const T* __restrict__ k, const T* __restrict__ v, T* kp, T* vp,
                                                      const int32_t* __restrict__ table,
                                                      const int32_t* __restrict__ lens,
                                                      const int32_t* __restrict__ count, int32_t* lens_out, int Hkv,
                                                      int Tn, int D, int P, int max_pages, int n_pages, int nchunk,
                                                      int limit) {
  const int b = (int)(blockIdx.x / ((int64_t)Hkv * nchunk));
  const int hc = (int)(blockIdx.x % ((int64_t)Hkv * nchunk));
  const int h = hc / nchunk, ch = hc % nchunk;
  const int len = lens[b];
  int cnt = count == nullptr ? Tn : count[b];
  cnt = cnt < 0 ? 0 : (cnt < Tn ? cnt : Tn);
  int ok = len >= 0 && len <= limit - cnt;   // (limit: at most max_pages * P)
  if (ok && cnt > 0) {
    const int p1 = (len + cnt - 1) / P;
    for (int p = len / P + threadIdx.x; p <= p1; p += 256) {
      const int page = table[(int64_t)b * max_pages + p];
      ok = ok && page >= 0 && page < n_pages;
    }
  }
  ok = __syncthreads_and(ok);
  if (hc == 0 && threadIdx.x == 0) lens_out[b] = ok ? len + cnt : len;
  if (!ok) return;
  const int t0 = ch * 64, t1 = cnt < t0 + 64 ? cnt : t0 + 64;
  constexpr int E = 16 / (int)sizeof(T);
  const int rv = D / E;                         // 16-byte pieces of a row
  for (int i = threadIdx.x; i < (t1 - t0) * rv; i += 256) {
    const int t = t0 + i / rv, d = (i % rv) * E;
    const int p = len + t, pi = p / P;
    const int64_t dst = (((int64_t)table[(int64_t)b * max_pages + pi] * Hkv + h) * P + (p - pi * P)) * D + d;
    const int64_t src = (((int64_t)b * Hkv + h) * Tn + t) * D + d;
    *reinterpret_cast<f32x4*>(kp + dst) = *reinterpret_cast<const f32x4*>(k + src);
    *reinterpret_cast<f32x4*>(vp + dst) = *reinterpret_cast<const f32x4*>(v + src);
  }
}

struct PagedPlan {
  int NT, HT, W;
  int64_t R;             // rows: sequences x KV heads x head tiles
  bool joined;           // there may be pieces to join
};
// Shares: two for every compute unit, so that one loads while the other starts
// or ends a piece (16 x 4K with a KV head for every head: 65 us, 82 with one);
// one where the rows are few and long (one sequence of 32K: 19.9 us, 20.9 with
// two; 32 of up to 32K: 215, 217).  Where the rows fill the chip and none can
// be long (1 MiB of keys and values), a workgroup takes a row instead (W = 0):
// nothing is counted and nothing joined (200 sequences of up to 900 at 12:2 heads
// of 64: 16.5 us, and 22.4 under a table of 32K positions, which takes shares).
static PagedPlan paged_plan(int B, int Hq, int Hkv, int row_bytes, int64_t cap, int cu) {
  PagedPlan p;
  const int G = Hq / Hkv;
  p.NT = G > 16 && row_bytes <= 256 ? 2 : 1;   // (two tiles of 512-byte rows do not fit the registers)
  p.HT = (G + 16 * p.NT - 1) / (16 * p.NT);
  p.R = (int64_t)B * Hkv * p.HT;
  const int64_t most = p.R * ((cap + kUnit - 1) / kUnit);
  const bool rows = cap <= kUnit || (p.R >= cu && cap * 2 * row_bytes <= (1 << 20));
  const int64_t shares = p.R <= cu / 2 && cap >= 32 * kUnit ? cu : 2LL * cu;
  p.W = rows ? 0 : (int)(most < shares ? most : shares);
  p.joined = !rows;
  return p;
}
static bool paged_shape_ok(int B, int Hq, int Hkv, int D, int P, int max_pages, int n_pages) {
  return B >= 0 && B <= 65536 && Hkv >= 1 && Hq >= Hkv && Hq % Hkv == 0 && Hq <= 4096 &&
         (D == 16 || D == 32 || D == 64 || D == 128) && P >= 16 && P % 16 == 0 && max_pages >= 1 && n_pages >= 1 &&
         (int64_t)max_pages * P <= (1 << 30) &&
         (int64_t)B * Hq * (((int64_t)max_pages * P + kUnit - 1) / kUnit) <= INT32_MAX;   // units are counted in 32 bits
}

template <typename T, int D>
static int paged_launch(const PagedArgs& a, const PagedPlan& p, hipStream_t s) {
  NSA_CHECK(p.R < (1 << 24) && (int64_t)a.B * a.Hq < (1 << 22), NSA_ERR_SHAPE);   // grids hold less than 2^32 threads
  const unsigned grid = (unsigned)(p.W > 0 ? p.W : p.R);
  if (p.NT == 1)
    k_paged<T, D, 1><<<grid, 256, 0, s>>>(a);
  else if constexpr (D * sizeof(T) <= 256)
    k_paged<T, D, 2><<<grid, 256, 0, s>>>(a);
  if (p.joined) {
    // few rows are many pieces each: sixteen waves a head
    if (p.R * 16 <= p.W)
      k_paged_join<T, D, 16><<<(unsigned)(a.B * a.Hq), 1024, 0, s>>>(a, p.NT);
    else
      k_paged_join<T, D, 4><<<(unsigned)(a.B * a.Hq), 256, 0, s>>>(a, p.NT);
  }
  return nsa_launch_status();
}
template <typename T>
static int paged_dim(const PagedArgs& a, const PagedPlan& p, int D, hipStream_t s) {
  switch (D) {
    case 16: return paged_launch<T, 16>(a, p, s);
    case 32: return paged_launch<T, 32>(a, p, s);
    case 64: return paged_launch<T, 64>(a, p, s);
    case 128: return paged_launch<T, 128>(a, p, s);
  }
  return NSA_ERR_SHAPE;
}

}  // namespace nsa

static size_t paged_ws_bytes(int D, const nsa::PagedPlan& p) {
  return p.joined ? (size_t)(p.W + p.R) * 16 * p.NT * (D * sizeof(float) + sizeof(float2)) + (size_t)p.R * sizeof(int2)
                  : 16;
}

extern "C" size_t nsa_paged_workspace(int B, int Hq, int Hkv, int D, int P, int max_pages, int dtype, void* stream) {
  using namespace nsa;
  if (!paged_shape_ok(B, Hq, Hkv, D, P, max_pages, 1) || (dtype != NSA_F32 && dtype != NSA_BF16)) return 0;
  return paged_ws_bytes(D, paged_plan(B, Hq, Hkv, D * (dtype == NSA_BF16 ? 2 : 4), (int64_t)max_pages * P,
                                      device_cu_count(static_cast<hipStream_t>(stream))));
}

static int paged_limit(int max_pages, int P, int max_len) {
  return max_len < max_pages * P ? max_len : max_pages * P;
}

extern "C" int nsa_paged_attend_max(const void* q, const void* k_new, const void* v_new, void* k_pages, void* v_pages,
                                    const int32_t* table, const int32_t* lens, int32_t* lens_out, void* out,
                                    float* lse, void* workspace, size_t workspace_bytes, int B, int Hq, int Hkv, int D,
                                    int P, int max_pages, int n_pages, int max_len, float scale, int dtype,
                                    void* stream) {
  using namespace nsa;
  NSA_CHECK(paged_shape_ok(B, Hq, Hkv, D, P, max_pages, n_pages) && max_len >= 0, NSA_ERR_SHAPE);
  NSA_CHECK(dtype == NSA_F32 || dtype == NSA_BF16, NSA_ERR_DTYPE);
  if (B == 0) return NSA_OK;
  NSA_CHECK(q != nullptr && k_pages != nullptr && v_pages != nullptr && table != nullptr && lens != nullptr &&
                out != nullptr, NSA_ERR_ARG);
  NSA_CHECK((k_new == nullptr) == (v_new == nullptr) && (k_new == nullptr) == (lens_out == nullptr) &&
                lens_out != lens, NSA_ERR_ARG);
  const hipStream_t s = static_cast<hipStream_t>(stream);
  const PagedPlan p =
      paged_plan(B, Hq, Hkv, D * (dtype == NSA_BF16 ? 2 : 4), (int64_t)max_pages * P, device_cu_count(s));
  PagedArgs a{q, k_new, v_new, k_pages, v_pages, table, lens, lens_out, out, lse, nullptr, nullptr, nullptr, B, Hq, Hkv,
              Hq / Hkv, p.HT, P, P / 16, max_pages, n_pages, p.W, paged_limit(max_pages, P, max_len), scale * kLog2e};
  if (p.joined) {
    NSA_CHECK(workspace != nullptr && workspace_bytes >= paged_ws_bytes(D, p), NSA_ERR_WORKSPACE);
    const size_t slots = (size_t)(p.W + p.R) * 16 * p.NT;
    a.part_o = static_cast<float*>(workspace);
    a.part_ml = reinterpret_cast<float2*>(a.part_o + slots * D);
    a.row_info = reinterpret_cast<int2*>(a.part_ml + slots);
  }
  return dtype == NSA_BF16 ? paged_dim<bf16>(a, p, D, s) : paged_dim<float>(a, p, D, s);
}

extern "C" int nsa_paged_attend(const void* q, const void* k_new, const void* v_new, void* k_pages, void* v_pages,
                                const int32_t* table, const int32_t* lens, int32_t* lens_out, void* out, float* lse,
                                void* workspace, size_t workspace_bytes, int B, int Hq, int Hkv, int D, int P,
                                int max_pages, int n_pages, float scale, int dtype, void* stream) {
  return nsa_paged_attend_max(q, k_new, v_new, k_pages, v_pages, table, lens, lens_out, out, lse, workspace,
                              workspace_bytes, B, Hq, Hkv, D, P, max_pages, n_pages, INT32_MAX, scale, dtype, stream);
}

extern "C" int nsa_paged_append_max(const void* k, const void* v, void* k_pages, void* v_pages, const int32_t* table,
                                    const int32_t* lens, const int32_t* count, int32_t* lens_out, int B, int Hkv,
                                    int T, int D, int P, int max_pages, int n_pages, int max_len, int dtype,
                                    void* stream) {
  using namespace nsa;
  NSA_CHECK(paged_shape_ok(B, Hkv, Hkv, D, P, max_pages, n_pages) && T >= 0 && max_len >= 0, NSA_ERR_SHAPE);
  NSA_CHECK(dtype == NSA_F32 || dtype == NSA_BF16, NSA_ERR_DTYPE);
  if (B == 0) return NSA_OK;
  NSA_CHECK(k_pages != nullptr && v_pages != nullptr && table != nullptr && lens != nullptr && lens_out != nullptr &&
                lens != lens_out && (T == 0 || (k != nullptr && v != nullptr)), NSA_ERR_ARG);
  const int nchunk = T > 64 ? (T + 63) / 64 : 1;
  const int64_t grid = (int64_t)B * Hkv * nchunk;
  NSA_CHECK(grid < (1 << 24), NSA_ERR_SHAPE);   // a grid holds less than 2^32 threads
  const hipStream_t s = static_cast<hipStream_t>(stream);
  const int limit = paged_limit(max_pages, P, max_len);
  if (dtype == NSA_BF16)
    k_paged_append<bf16><<<(unsigned)grid, 256, 0, s>>>(
        static_cast<const bf16*>(k), static_cast<const bf16*>(v), static_cast<bf16*>(k_pages),
        static_cast<bf16*>(v_pages), table, lens, count, lens_out, Hkv, T, D, P, max_pages, n_pages, nchunk,
        limit);
  else
    k_paged_append<float><<<(unsigned)grid, 256, 0, s>>>(
        static_cast<const float*>(k), static_cast<const float*>(v), static_cast<float*>(k_pages),
        static_cast<float*>(v_pages), table, lens, count, lens_out, Hkv, T, D, P, max_pages, n_pages, nchunk,
        limit);
  return nsa_launch_status();
}

extern "C" int nsa_paged_append(const void* k, const void* v, void* k_pages, void* v_pages, const int32_t* table,
                                const int32_t* lens, const int32_t* count, int32_t* lens_out, int B, int Hkv, int T,
                                int D, int P, int max_pages, int n_pages, int dtype, void* stream) {
  return nsa_paged_append_max(k, v, k_pages, v_pages, table, lens, count, lens_out, B, Hkv, T, D, P, max_pages,
                              n_pages, INT32_MAX, dtype, stream);
}
