// Attention of one new token of every sequence over a paged key-value cache,
// with the append of its key and value rows, and the writing of whole prompts.
//
//   pages  [n_pages][Hkv][P][D]  keys and values; P a multiple of 16
//   table  [B][max_pages]        position p of sequence b lies in page table[b][p / P], row p % P
//   lens   [B]                   keys of each sequence before the step
//   out[b][h] = softmax(scale q K^T) V over the keys 0 .. n-1 of KV head h / (Hq / Hkv)
//
// A step is bound by reading each key and value row once.  A workgroup of four
// waves takes a chunk of one sequence's keys for one KV head (and up to 32 of
// its query heads); each wave takes tiles of 32 keys in turn, with the running
// maximum and sum of the softmax, and the four are joined in LDS.  With more
// than one chunk the unnormalised outputs go to the workspace and a second
// launch joins them.
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
// Rows at and past a sequence's length are never read: they may hold anything.
// The step's own row is read from the caller's new rows, not from the page it
// is written to, so that no read waits for that write.
#include "nsa_launch.h"
#include "nsa_paged_index.h"
#include "nsa_tiles.h"

namespace nsa {

struct PagedArgs {
  const void *q, *k_new, *v_new;     // [B][Hq][D], [B][Hkv][D] (null: no append)
  void *kp, *vp;
  const int32_t *table, *lens;
  int32_t* lens_out;                 // or null
  void* out;
  float* lse;                        // or null
  float* part_o;                     // [B][Hq][nsp][D]
  float2* part_ml;                   // [B][Hq][nsp]
  int B, Hq, Hkv, G, HT, P, rpp;     // HT: head tiles of a KV head; rpp: runs of 16 in a page
  int max_pages, n_pages, nsp, chunk;
  float sl2;                         // scale * log2 e
};

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

// K operands and V rows of one tile of 32 keys
template <typename T, int D> struct KVTile {
  Frag<T> k[2][Dims<D>::KC];
  VRun<T, D / 16> v[8];
};

// NT: tiles of 16 query heads.
template <typename T, int D, int NT>
__global__ __launch_bounds__(256) void k_paged(const PagedArgs a) {
  constexpr int KC = Dims<D>::KC, DT = Dims<D>::DT, VL = D / 16;
  constexpr bool SPLIT_P = sizeof(T) == 2;
  const int lane = threadIdx.x & 63, g = lane >> 4, c = lane & 15;
  const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  int64_t bid = blockIdx.x;
  const int sp = (int)(bid % a.nsp);
  bid /= a.nsp;
  const int ht = (int)(bid % a.HT);
  bid /= a.HT;
  const int hkv = (int)(bid % a.Hkv), b = (int)(bid / a.Hkv);

  const int cap = a.max_pages * a.P;
  const int len = a.lens[b];
  int n = len < 0 ? 0 : (len < cap ? len : cap);     // keys attended
  int pos = -1;                                      // the appended row's position
  if (a.k_new != nullptr) {
    pos = paged_new_pos(a.table + (int64_t)b * a.max_pages, len, a.P, a.max_pages, a.n_pages);
    if (pos >= 0) n = len + 1;
  }
  if (a.lens_out != nullptr && sp == 0 && ht == 0 && hkv == 0 && threadIdx.x == 0) a.lens_out[b] = pos >= 0 ? n : len;
  const int c0 = sp * a.chunk;
  const int c1 = n < c0 + a.chunk ? n : c0 + a.chunk;
  if (c0 >= c1 && sp > 0) return;                    // (uniform; part 0 of an empty sequence writes its zeros)

  const T* kp = static_cast<const T*>(a.kp);
  const T* vp = static_cast<const T*>(a.vp);
  const T* kn = static_cast<const T*>(a.k_new) + ((int64_t)b * a.Hkv + hkv) * D;
  const T* vn = static_cast<const T*>(a.v_new) + ((int64_t)b * a.Hkv + hkv) * D;

  // the append: one wave of the first head tile whose chunk holds the position
  if (pos >= c0 && pos < c1 && ht == 0 && w == 0) {
    const int64_t at = run_base(a, b, hkv, pos >> 4, D) + (int64_t)(pos & 15) * D;
    for (int d = lane; d < D; d += 64) {
      static_cast<T*>(a.kp)[at + d] = kn[d];
      static_cast<T*>(a.vp)[at + d] = vn[d];
    }
  }

  Frag<T> qf[NT][KC];
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) {
    const int hg = ht * 16 * NT + 16 * nt + c;
    const T* row = hg < a.G ? static_cast<const T*>(a.q) + ((int64_t)b * a.Hq + (int64_t)hkv * a.G + hg) * D : nullptr;
    load_row_frags<T, D>(qf[nt], row, g);
  }
  FwdAcc<D> acc[NT];
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) acc[nt].init();

  // this wave's tiles: 32 keys every 128; lane i looks up run i of them
  const int my0 = c0 + 32 * w;
  const int ntile = c1 > my0 ? (c1 - my0 + 127) / 128 : 0;
  int64_t base = -1;
  {
    const int key = my0 + 128 * (lane >> 1) + 16 * (lane & 1);
    if ((lane >> 1) < ntile && key < c1) base = run_base(a, b, hkv, key >> 4, D);
  }
  const int kofs0 = ((8 * (c >> 2)) & 15) + (c & 3);
  for (int i = 0; i < ntile; ++i) {
    const int kb = my0 + 128 * i;
    const int64_t b0 = __shfl(base, 2 * i, 64), b1 = __shfl(base, 2 * i + 1, 64);
    KVTile<T, D> t;
    const int64_t bk = c >= 8 ? b1 : b0, bv = g >= 2 ? b1 : b0;
    // keys of this tile that this lane's K rows (m) and V rows may be read for
    const bool whole = kb + 32 <= c1 && b0 >= 0 && b1 >= 0 && !(pos >= kb && pos < kb + 32);
    if (whole) {
#pragma unroll
      for (int mt = 0; mt < 2; ++mt)
#pragma unroll
        for (int kc = 0; kc < KC; ++kc) {
          if (32 * kc + 8 * g < D)
            t.k[mt][kc].load(kp + bk + (kofs0 + 4 * mt) * D + 32 * kc + 8 * g);
          else
            t.k[mt][kc].zero();
        }
#pragma unroll
      for (int j = 0; j < 8; ++j) t.v[j] = vrun_load<T, VL>(vp + bv + (((8 * g) & 15) + j) * D + VL * c);
    } else {
#pragma unroll
      for (int mt = 0; mt < 2; ++mt) {
        const int key = kb + 8 * (c >> 2) + 4 * mt + (c & 3);
        const T* row = key == pos ? kn : (key < c1 && bk >= 0 ? kp + bk + (kofs0 + 4 * mt) * D : nullptr);
#pragma unroll
        for (int kc = 0; kc < KC; ++kc) {
          if (row != nullptr && 32 * kc + 8 * g < D)
            t.k[mt][kc].load(row + 32 * kc + 8 * g);
          else
            t.k[mt][kc].zero();
        }
      }
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const int key = kb + 8 * g + j;
        const T* row = key == pos ? vn : (key < c1 && bv >= 0 ? vp + bv + (((8 * g) & 15) + j) * D : nullptr);
        t.v[j] = row != nullptr ? vrun_load<T, VL>(row + VL * c) : vrun_zero<T, VL>();
      }
    }
    // visible keys kb + 8 g .. + 7 of this lane
    const uint32_t vm = bv >= 0 ? range_mask(kb + 8 * g, 0, c1 - 1) : 0u;
    Frag<T> vf[DT];
#pragma unroll
    for (int dt = 0; dt < DT; ++dt) {
      if constexpr (sizeof(T) == 2) {
#pragma unroll
        for (int j = 0; j < 8; ++j) vf[dt].v[j] = vrun_elem<T, VL>(t.v[j], dt);
      } else {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          vf[dt].lo[j] = vrun_elem<T, VL>(t.v[j], dt);
          vf[dt].hi[j] = vrun_elem<T, VL>(t.v[4 + j], dt);
        }
      }
    }
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      FwdAcc<D>& A = acc[nt];
      f32x4 s0 = zero4(), s1 = zero4();
#pragma unroll
      for (int kc = 0; kc < KC; ++kc) {
        mma(s0, t.k[0][kc], qf[nt][kc]);
        mma(s1, t.k[1][kc], qf[nt][kc]);
      }
      float sv[8] = {s0[0], s0[1], s0[2], s0[3], s1[0], s1[1], s1[2], s1[3]};
      float mx = kMaskScore;
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        sv[j] = ((vm >> j) & 1u) ? sv[j] * a.sl2 : kMaskScore;
        mx = fmaxf(mx, sv[j]);
      }
      mx = group4_max(mx);
      const float mn = fmaxf(A.m, mx);
      const float alpha = fast_exp2(A.m - mn);
      float p[8], ps = 0.0f;
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        p[j] = ((vm >> j) & 1u) ? fast_exp2(sv[j] - mn) : 0.0f;
        ps += p[j];
      }
      A.l = A.l * alpha + ps;
      A.m = mn;
#pragma unroll
      for (int dt = 0; dt < DT; ++dt) A.o[dt] *= alpha;
      Frag<T> pf;
      pf.set(p);
#pragma unroll
      for (int dt = 0; dt < DT; ++dt) mma(A.o[dt], vf[dt], pf);
      if constexpr (SPLIT_P) {
#pragma unroll
        for (int j = 0; j < 8; ++j) p[j] -= (float)pf.elem(j);
        pf.set(p);
#pragma unroll
        for (int dt = 0; dt < DT; ++dt) mma(A.o[dt], vf[dt], pf);
      }
    }
  }

  // join the four waves: their outputs against the common maximum, added in wave order
  __shared__ float so[16][D + 4];
  __shared__ float sm[4][16], sl[4][16];
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) {
    FwdAcc<D>& A = acc[nt];
    A.l = group4_sum(A.l);
    if (nt > 0) __syncthreads();
    if (g == 0) sm[w][c] = A.m, sl[w][c] = A.l;
    __syncthreads();
    const float m = fmaxf(fmaxf(sm[0][c], sm[1][c]), fmaxf(sm[2][c], sm[3][c]));
    float l = 0.0f;
#pragma unroll
    for (int i = 0; i < 4; ++i) l += sl[i][c] * fast_exp2(sm[i][c] - m);
    const float f = fast_exp2(A.m - m);
    for (int i = 0; i < 4; ++i) {
      if (i == w) {
#pragma unroll
        for (int r = 0; r < 4; ++r)
#pragma unroll
          for (int dt = 0; dt < DT; ++dt) {
            float* p = &so[c][VL * (4 * g + r) + dt];
            const float v = A.o[dt][r] * f;
            *p = i == 0 ? v : *p + v;
          }
      }
      __syncthreads();
    }
    // 16 threads a head
    const int hr = threadIdx.x >> 4, x = threadIdx.x & 15;
    const int hg = ht * 16 * NT + 16 * nt + hr;
    const float lt = __shfl(l, hr & 15, 64), mt = __shfl(m, hr & 15, 64);   // (lane hr of each wave holds column hr)
    if (hg < a.G) {
      const int64_t head = (int64_t)b * a.Hq + (int64_t)hkv * a.G + hg;
      if (a.nsp == 1) {
        const float inv = lt > 0.0f ? 1.0f / lt : 0.0f;
        T* out = static_cast<T*>(a.out) + head * D;
        for (int d = x; d < D; d += 16) out[d] = (T)(lt > 0.0f ? so[hr][d] * inv : so[hr][d] * 0.0f);
        if (a.lse != nullptr && x == 0) a.lse[head] = lt > 0.0f ? (mt + __log2f(lt)) * kLn2 : (lt == 0.0f ? kLseEmpty : lt);
      } else {
        float* out = a.part_o + (head * a.nsp + sp) * D;
        for (int d = x; d < D; d += 16) out[d] = so[hr][d];
        if (x == 0) a.part_ml[head * a.nsp + sp] = make_float2(mt, lt);
      }
    }
  }
}

// Joins a head's parts: one workgroup of four waves; the waves take parts in turn.
template <typename T, int D>
__global__ __launch_bounds__(256) void k_paged_join(const PagedArgs a) {
  __shared__ float so[4][D], sl[4];
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
  const int64_t head = blockIdx.x;
  const int b = (int)(head / a.Hq);
  const int cap = a.max_pages * a.P;
  const int len = a.lens_out != nullptr ? a.lens_out[b] : a.lens[b];
  const int n = len < 0 ? 0 : (len < cap ? len : cap);
  int np = (n + a.chunk - 1) / a.chunk;
  np = np < 1 ? 1 : np;
  const float2* ml = a.part_ml + head * a.nsp;
  const float* po = a.part_o + head * a.nsp * D;
  float m = kMaskScore;
  for (int i = lane; i < np; i += 64) m = fmaxf(m, ml[i].x);
#pragma unroll
  for (int x = 1; x < 64; x <<= 1) m = xor_max(m, x);
  constexpr int E = D >= 64 ? D / 64 : 1;
  float o[E], l = 0.0f;
#pragma unroll
  for (int e = 0; e < E; ++e) o[e] = 0.0f;
#pragma unroll 4
  for (int i = w; i < np; i += 4) {
    const float2 s = ml[i];
    const float f = fast_exp2(s.x - m);
    l += s.y * f;
#pragma unroll
    for (int e = 0; e < E; ++e)
      if (E * lane + e < D) o[e] += po[(int64_t)i * D + E * lane + e] * f;
  }
#pragma unroll
  for (int e = 0; e < E; ++e)
    if (E * lane + e < D) so[w][E * lane + e] = o[e];
  if (lane == 0) sl[w] = l;
  __syncthreads();
  l = ((sl[0] + sl[1]) + sl[2]) + sl[3];
  const float inv = l > 0.0f ? 1.0f / l : 0.0f;
  if ((int)threadIdx.x < D) {
    const int d = threadIdx.x;
    const float v = ((so[0][d] + so[1][d]) + so[2][d]) + so[3][d];
    static_cast<T*>(a.out)[head * D + d] = (T)(v * inv);
  }
  if (a.lse != nullptr && threadIdx.x == 0) a.lse[head] = l > 0.0f ? (m + __log2f(l)) * kLn2 : (l == 0.0f ? kLseEmpty : l);
}

// Rows [B][Hkv][Tn][D] to positions lens[b] .. lens[b] + count[b] - 1: all of a
// sequence's rows, or none where they do not all have a page.
template <typename T>
__global__ __launch_bounds__(256) void k_paged_append(const T* __restrict__ k, const T* __restrict__ v, T* kp, T* vp,
                                                      const int32_t* __restrict__ table,
                                                      const int32_t* __restrict__ lens,
                                                      const int32_t* __restrict__ count, int32_t* lens_out, int Hkv,
                                                      int Tn, int D, int P, int max_pages, int n_pages, int nchunk) {
  const int b = (int)(blockIdx.x / ((int64_t)Hkv * nchunk));
  const int hc = (int)(blockIdx.x % ((int64_t)Hkv * nchunk));
  const int h = hc / nchunk, ch = hc % nchunk;
  const int cap = max_pages * P;
  const int len = lens[b];
  int cnt = count == nullptr ? Tn : count[b];
  cnt = cnt < 0 ? 0 : (cnt < Tn ? cnt : Tn);
  int ok = len >= 0 && len <= cap - cnt;
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
  int NT, HT, chunk, nsp;
};
// Chunk: as long as leaves four workgroups for every compute unit (fewer
// parts to join), from 128 keys (a tile for each wave) to 2048.
static PagedPlan paged_plan(int B, int Hq, int Hkv, int D, int64_t cap, int cu) {
  PagedPlan p;
  const int G = Hq / Hkv;
  p.NT = G > 16 ? 2 : 1;
  p.HT = (G + 16 * p.NT - 1) / (16 * p.NT);
  const int64_t rows = (int64_t)B * Hkv * p.HT;
  p.chunk = 2048;
  while (p.chunk > 128 && rows * ((cap + p.chunk - 1) / p.chunk) < 4LL * cu) p.chunk /= 2;
  p.nsp = (int)((cap + p.chunk - 1) / p.chunk);
  return p;
}
static bool paged_shape_ok(int B, int Hq, int Hkv, int D, int P, int max_pages, int n_pages) {
  return B >= 0 && B <= 65536 && Hkv >= 1 && Hq >= Hkv && Hq % Hkv == 0 && Hq <= 4096 &&
         (D == 16 || D == 32 || D == 64 || D == 128) && P >= 16 && P % 16 == 0 && max_pages >= 1 && n_pages >= 1 &&
         (int64_t)max_pages * P <= (1 << 30);
}

template <typename T, int D>
static int paged_launch(const PagedArgs& a, int NT, hipStream_t s) {
  const int64_t grid = (int64_t)a.B * a.Hkv * a.HT * a.nsp;
  NSA_CHECK(grid <= 0x7fffffffLL, NSA_ERR_SHAPE);
  if (NT == 2)
    k_paged<T, D, 2><<<(unsigned)grid, 256, 0, s>>>(a);
  else
    k_paged<T, D, 1><<<(unsigned)grid, 256, 0, s>>>(a);
  if (a.nsp > 1) k_paged_join<T, D><<<(unsigned)(a.B * a.Hq), 256, 0, s>>>(a);
  return nsa_launch_status();
}
template <typename T>
static int paged_dim(const PagedArgs& a, int NT, int D, hipStream_t s) {
  switch (D) {
    case 16: return paged_launch<T, 16>(a, NT, s);
    case 32: return paged_launch<T, 32>(a, NT, s);
    case 64: return paged_launch<T, 64>(a, NT, s);
    case 128: return paged_launch<T, 128>(a, NT, s);
  }
  return NSA_ERR_SHAPE;
}

}  // namespace nsa

extern "C" size_t nsa_paged_workspace(int B, int Hq, int Hkv, int D, int P, int max_pages, void* stream) {
  using namespace nsa;
  if (!paged_shape_ok(B, Hq, Hkv, D, P, max_pages, 1)) return 0;
  const PagedPlan p = paged_plan(B, Hq, Hkv, D, (int64_t)max_pages * P, device_cu_count(static_cast<hipStream_t>(stream)));
  return p.nsp == 1 ? 16 : (size_t)B * Hq * p.nsp * (D * sizeof(float) + sizeof(float2)) + 16;
}

extern "C" int nsa_paged_attend(const void* q, const void* k_new, const void* v_new, void* k_pages, void* v_pages,
                                const int32_t* table, const int32_t* lens, int32_t* lens_out, void* out, float* lse,
                                void* workspace, size_t workspace_bytes, int B, int Hq, int Hkv, int D, int P,
                                int max_pages, int n_pages, float scale, int dtype, void* stream) {
  using namespace nsa;
  NSA_CHECK(paged_shape_ok(B, Hq, Hkv, D, P, max_pages, n_pages), NSA_ERR_SHAPE);
  NSA_CHECK(dtype == NSA_F32 || dtype == NSA_BF16, NSA_ERR_DTYPE);
  if (B == 0) return NSA_OK;
  NSA_CHECK(q != nullptr && k_pages != nullptr && v_pages != nullptr && table != nullptr && lens != nullptr &&
                out != nullptr, NSA_ERR_ARG);
  NSA_CHECK((k_new == nullptr) == (v_new == nullptr) && (k_new == nullptr) == (lens_out == nullptr) &&
                lens_out != lens, NSA_ERR_ARG);
  const hipStream_t s = static_cast<hipStream_t>(stream);
  const PagedPlan p = paged_plan(B, Hq, Hkv, D, (int64_t)max_pages * P, device_cu_count(s));
  PagedArgs a{q, k_new, v_new, k_pages, v_pages, table, lens, lens_out, out, lse, nullptr, nullptr, B, Hq, Hkv,
              Hq / Hkv, p.HT, P, P / 16, max_pages, n_pages, p.nsp, p.chunk, scale * kLog2e};
  if (p.nsp > 1) {
    NSA_CHECK(workspace != nullptr && workspace_bytes >= nsa_paged_workspace(B, Hq, Hkv, D, P, max_pages, stream),
              NSA_ERR_WORKSPACE);
    a.part_o = static_cast<float*>(workspace);
    a.part_ml = reinterpret_cast<float2*>(a.part_o + (size_t)B * Hq * p.nsp * D);
  }
  return dtype == NSA_BF16 ? paged_dim<bf16>(a, p.NT, D, s) : paged_dim<float>(a, p.NT, D, s);
}

extern "C" int nsa_paged_append(const void* k, const void* v, void* k_pages, void* v_pages, const int32_t* table,
                                const int32_t* lens, const int32_t* count, int32_t* lens_out, int B, int Hkv, int T,
                                int D, int P, int max_pages, int n_pages, int dtype, void* stream) {
  using namespace nsa;
  NSA_CHECK(paged_shape_ok(B, Hkv, Hkv, D, P, max_pages, n_pages) && T >= 0, NSA_ERR_SHAPE);
  NSA_CHECK(dtype == NSA_F32 || dtype == NSA_BF16, NSA_ERR_DTYPE);
  if (B == 0) return NSA_OK;
  NSA_CHECK(k_pages != nullptr && v_pages != nullptr && table != nullptr && lens != nullptr && lens_out != nullptr &&
                lens != lens_out && (T == 0 || (k != nullptr && v != nullptr)), NSA_ERR_ARG);
  const int nchunk = T > 64 ? (T + 63) / 64 : 1;
  const int64_t grid = (int64_t)B * Hkv * nchunk;
  NSA_CHECK(grid <= 0x7fffffffLL, NSA_ERR_SHAPE);
  const hipStream_t s = static_cast<hipStream_t>(stream);
  if (dtype == NSA_BF16)
    k_paged_append<bf16><<<(unsigned)grid, 256, 0, s>>>(
        static_cast<const bf16*>(k), static_cast<const bf16*>(v), static_cast<bf16*>(k_pages),
        static_cast<bf16*>(v_pages), table, lens, count, lens_out, Hkv, T, D, P, max_pages, n_pages, nchunk);
  else
    k_paged_append<float><<<(unsigned)grid, 256, 0, s>>>(
        static_cast<const float*>(k), static_cast<const float*>(v), static_cast<float*>(k_pages),
        static_cast<float*>(v_pages), table, lens, count, lens_out, Hkv, T, D, P, max_pages, n_pages, nchunk);
  return nsa_launch_status();
}
