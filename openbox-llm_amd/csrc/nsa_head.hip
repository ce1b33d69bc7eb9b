// Log probabilities of tokens from the rows behind the last norm, without the
// logits.  x [N][D], W [V][D]; z = x W^T exists only as tiles in registers:
//
//   lse_n = ln sum_v e^{z_nv},   logp_n = x_n . W_{t_n} - lse_n   (0 where t_n is no token)
//
// and with a_n = dlse_n - dlogp_n, b_n = dlogp_n (both without dlogp where t_n is none)
//
//   dz_nv = a_n e^{z_nv - lse_n} + b_n [v = t_n],   dx = dz W,   dW = dz^T x.
//
// Four products on the matrix instructions with float32 sums (bf16: 32x32x16): z for the
// log sums (a running maximum and sum in registers), z again for dz, and the two
// of the gradients.  dz exists for a piece of the vocabulary at a time; beside float32 rows it
// is float32 or its planes, beside bf16 rows it is rounded once to bf16 as the products'
// operand.  Most of both gradients is the target's own element, whose rounding no sum
// averages: what it leaves, rest_n, goes to the results in float32, as rest_n W_{t_n} to
// dx and, summed over a token's rows, as rest_n x_n to dW.  (Root of the squares' sum, 40 cases of 1 to
// 19900 rows and 128 to 183000 tokens: both gradients are 1.00 times as far off 64 bits as their
// rounding to bf16 makes them, 1.16 at most; 1.36 and up to 1.8 without the rests. 1 to 2% of the time of large calls.)
//
// float32 rows and weights of few rows go through v_mfma_f32_32x32x2_f32 as they are; of many
// as three bf16 planes p0 + p1 + p2 = x, |x - p0 - p1 - p2| <= 2^-27 |x|: six products of
// planes (i + j <= 2) leave out terms below 2^-26 of the product, less than float32's own
// rounding.  A bf16 operand beside float32 rows is one plane; float32 weights beside bf16 rows
// are rounded to bf16 first.
//
// Layout: an operand is read either along its rows (the contraction runs along
// memory) into a [rows][64] tile, or across them into a [64][columns] tile that
// the transposed LDS reads turn; no transposed copy is made.  Results have the
// 32-row tile's rows permuted (perm32), so that a lane holds eight neighbouring
// elements of an output row.
//
// Large products are bound by the matrix unit: 32768 x 32000 x d768 in bf16, 1.61 TFLOP a
// product: z with its log sums 1.33 to 1.41 ms (1140 to 1210 TFLOP/s), dz 1.64 to 1.73 with
// its exponentials and 2.1 GB of stores, dx and dW 1.40 each (1150); a library product of these
// shapes takes 1.45 (z), 1.47 (dx) and 2.00 (dW).  At d4096 (8192 x 8192) all four run at
// 1310.  Few rows are bound by W: 32 x 32000 x d768 reads its 49 MB in 11 us.
#include "nsa_launch.h"
#include "nsa_rows.h"
#include "nsa_tile32.h"

namespace nsa {

constexpr int64_t kHeadRows = 1 << 22;       // most rows of x
constexpr int kHeadVocab = 1 << 24;
constexpr int kHeadWide = 1 << 16;           // widest row
constexpr size_t kHeadPiece = 1u << 30;      // bytes of dz held at a time: the backward of 32768 x 32000 x d768 takes
                                             // 4.55 ms, 5.03 with half of them (the parts of dx and more partial
                                             // rounds), 4.36 in one piece
constexpr int64_t kHeadPieceMost = 1 << 20;  // most tokens of a piece: offsets within a stage have 32 bits

// An operand of a product: bf16 planes; ROWS: [rows][ld], contraction along a row;
// otherwise [contraction][ld].
struct HeadOperand {
  const void* p;   // bf16, or float32 where the shape's elements are
  int64_t plane;   // elements between planes
  int64_t ld;      // elements between rows, a multiple of 8
  int rows;        // rows (ROWS) or columns: of the result
  int k_rows;      // not ROWS: contraction elements that exist in memory (at least K)
};

// One product C[m][n] = sum over plane pairs and k < K of A[m][k] B[n][k].
struct HeadProduct {
  HeadOperand a, b;
  int K;
  int pa, pb;      // planes
};

// Plane pairs (of a, of b) in the order they are added, the small ones first.  The
// rows' side b has three planes where a has.
__device__ __forceinline__ int head_pairs(int pa, int pb) { return pb == 1 ? 1 : pa == 1 ? 3 : 6; }
__device__ __forceinline__ void head_pair(int pa, int pb, int i, int& x, int& y) {
  if (pb == 1) {
    x = y = 0;
  } else if (pa == 1) {   // (0,2) (0,1) (0,0)
    x = 0;
    y = 2 - i;
  } else {                // (2,0) (1,1) (0,2) (1,0) (0,1) (0,0)
    x = i == 0 ? 2 : i == 1 || i == 3 ? 1 : 0;
    y = i == 2 ? 2 : i == 1 || i == 4 ? 1 : 0;
  }
}

// What a product's operands are made of.  A step of the contraction is 128 bytes of a
// row; a fragment is 16 bytes a lane: 8 elements of bf16 for one matrix instruction,
// 4 of float32 for four.
template <typename E> struct HeadType;
template <> struct HeadType<bf16> {
  typedef bf16x8 Frag;
  static __device__ __forceinline__ f32x16 product(Frag a, Frag b, f32x16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
  }
};
template <> struct HeadType<float> {
  typedef f32x4 Frag;
  static __device__ __forceinline__ f32x16 product(Frag a, Frag b, f32x16 c) {
#pragma unroll
    for (int j = 0; j < 4; ++j) c = __builtin_amdgcn_mfma_f32_32x32x2f32(a[j], b[j], c, 0, 0, 0);
    return c;
  }
};

// A stage of one operand: T rows (ROWS) or columns x kStep contraction elements, in
// 16-byte chunks.  Chunks are swizzled so that 16 neighbouring lanes' 16-byte reads, the
// transposed reads' 32-byte pieces of four rows, or 32 neighbouring columns of two rows
// meet every bank once.
template <typename E, int T, int kThreads, bool ROWS>
struct HeadTile {
  typedef typename HeadType<E>::Frag Frag;
  static constexpr bool kWide = sizeof(E) == 4;
  static constexpr int kB = sizeof(E), kChunk = 16 / kB, kStep = 128 / kB, kBytes = T * 128;
  static constexpr int kLoads = kBytes / 16 / kThreads;   // requests a thread, kThreads chunks each
  static constexpr int kCpr = ROWS ? 8 : T / kChunk;      // chunks a row of the stage
  static constexpr int kRows = kThreads / kCpr;           // rows of the stage a request
  static_assert(kBytes % (16 * kThreads) == 0 && (ROWS || T >= 128), "a tile of whole requests");
  static __device__ __forceinline__ int key(int r) {
    return ROWS ? (r >> 1) & 7 : kWide ? 8 * ((r >> 2) & 1) : 4 * (r & 3) + ((r >> 2) & 3);
  }

  // Request j brings rows j kRows + tid / kCpr of the stage, each lane 16 bytes.  Past
  // the operand its last row (first column) is read: what is past the result's last row
  // (column) is never stored, and past the contraction's end one of the two operands
  // (packed rows, dz) has zeros in memory up to a whole stage.
  uint32_t off[kLoads];   // bytes from the stage's base
  uint64_t base;          // the next stage's rows (columns) `first` .., elements k ..: wave-uniform
  int first, left;        // left: contraction elements from k on that exist
  __device__ __forceinline__ void place(const HeadOperand& o, int tid) {
    const int last = o.rows - 1 - first, end = left - 1;   // >= 0
#pragma unroll
    for (int j = 0; j < kLoads; ++j) {
      const int r = j * kRows + tid / kCpr, c = (tid % kCpr) ^ key(r);
      if (ROWS)
        off[j] = (uint32_t)((r < last ? r : last) * o.ld * kB + c * 16);
      else
        off[j] = (uint32_t)((r < end ? r : end) * o.ld * kB + (kChunk * c <= last ? c * 16 : 0));
    }
  }
  __device__ __forceinline__ void aim(const HeadOperand& o, int first_, int pl, int k, int tid) {
    first = first_;
    left = o.k_rows - k;
    const E* p = static_cast<const E*>(o.p) + pl * o.plane + (ROWS ? (int64_t)first * o.ld + k : (int64_t)k * o.ld + first);
    base = (uint64_t)(uintptr_t)p;
    base = u64_from_halves(__builtin_amdgcn_readfirstlane((uint32_t)base),
                           __builtin_amdgcn_readfirstlane((uint32_t)(base >> 32)));
    place(o, tid);
  }
  __device__ __forceinline__ void next(const HeadOperand& o, int tid) {
    left -= kStep;
    base += ROWS ? 128 : (uint64_t)o.ld * 128;
    if (!ROWS && left < kStep) place(o, tid);
  }
  // Request J of a stage; lds: the wave's place in it.
  template <int J>
  __device__ __forceinline__ void request(uint32_t lds) const {
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2" ::"s"(lds + J * kThreads * 16), "v"(off[J]),
                 "s"(base)
                 : "memory", "m0");
  }
  // Fragments of a wave: of the 32-row tile i from row w0 on (a multiple of 32, of 32 MT
  // where there are MT and not ROWS), row m (PERM: perm32(m)), 16 bytes of the contraction
  // from chunk 2 s + h of the step on.  `at` is the lane's byte address in LDS (stages lie on
  // 16 KB) for i = s = 0; i and s enter by addition, or by exclusive or where the swizzle has their bits.
  template <bool PERM>
  static __device__ __forceinline__ uint32_t lane_at(int w0, int lane) {
    const int m = PERM ? perm32(lane & 31) : lane & 31, h = lane >> 5;
    if (ROWS) return (uint32_t)((w0 + m) * 128 + ((h ^ key(m)) << 4));
    if (kWide) {
      const int col = w0 + m;
      return (uint32_t)(4 * h * T * 4 + (((col >> 2) ^ key(4 * h)) << 4) + (col & 3) * 4);
    }
    const int g = lane >> 4, r = 8 * (g >> 1) + ((lane >> 2) & 3);
    int q = lane & 3;
    if (PERM) q = ((q & 1) << 1) | (q >> 1);   // perm32 swaps bits 2 and 3 of the row
    const int col = w0 + 16 * (g & 1) + 4 * q;
    return (uint32_t)(r * T * 2 + (((col >> 3) ^ key(r)) << 4) + (col & 7) * 2);
  }
  static __device__ __forceinline__ Frag frag(uint32_t at, int i, int s) {
#define NSA_LDS(type, a) ((__attribute__((address_space(3))) type*)(uintptr_t)(a))
    if constexpr (ROWS) {
      return *NSA_LDS(Frag, (at ^ (32 * s)) + 32 * i * 128);
    } else if constexpr (kWide) {
      Frag f;
#pragma unroll
      for (int j = 0; j < 4; ++j) f[j] = *NSA_LDS(float, (at ^ (128 * i)) + (8 * s + j) * T * 4);
      return f;
    } else {
      typedef short s16x8 __attribute__((ext_vector_type(8)));
      const uint32_t a0 = at ^ (64 * i), a1 = a0 ^ 16;   // (rows r + 4: another key by 1)
      const s16x4 u = __builtin_amdgcn_ds_read_tr16_b64_v4i16(NSA_LDS(s16x4, a0 + 16 * s * T * 2));
      const s16x4 v = __builtin_amdgcn_ds_read_tr16_b64_v4i16(NSA_LDS(s16x4, a1 + (16 * s + 4) * T * 2));
#undef NSA_LDS
      const s16x8 f = (s16x8){u[0], u[1], u[2], u[3], v[0], v[1], v[2], v[3]};
      return __builtin_bit_cast(bf16x8, f);
    }
  }
};

// Tile shape: TM x TN of the result over WM x WN waves, NS stages, kPerCu workgroups a CU.
template <int TM_, int TN_, int WM_, int WN_, int NS_, int PER_CU_, typename E_ = bf16>
struct HeadShape {
  typedef E_ E;
  static constexpr int TM = TM_, TN = TN_, WM = WM_, WN = WN_, NS = NS_, kStep = 128 / (int)sizeof(E), kPerCu = PER_CU_;
  static constexpr int kThreads = WM * WN * 64, kPerSimd = kPerCu * WM * WN / 4;   // waves a SIMD
  static constexpr int MT = TM / WM / 32, NT = TN / WN / 32;   // 32 x 32 tiles of a wave
  static_assert(WM * WN % 4 == 0 && MT >= 1 && NT >= 1 && NS >= 2, "whole waves a SIMD");
};

// What a workgroup computes: tiles (m, n) of the result, each over the steps q0 .. q1 - 1
// of its contraction (a step: kStep elements of one plane pair; pairs one after another).
struct HeadSpan {
  int m, n, q0, q1;
};
template <class S>
__device__ __forceinline__ int head_steps(const HeadProduct& pr) {
  return head_pairs(pr.pa, pr.pb) * ((pr.K + S::kStep - 1) / S::kStep);
}

// f(I), f(I + 1), .. f(N - 1) with constants
template <int I, int N, typename F>
__device__ __forceinline__ void head_range(F&& f) {
  if constexpr (I < N) {
    f(std::integral_constant<int, I>{});
    head_range<I + 1, N>(f);
  }
}

// The spans i = 0 .. spans - 1, `total` steps in all; done(span, wm, wn, acc) takes each result,
// begin(span, wn) may ask for what that needs.
//
// All steps of all spans are one pipeline of NS stages in LDS.  One or two waves a SIMD leave
// the matrix unit idle wherever more than a few other instructions stand between two
// products, so that everything else is spread: a wave reads the fragments of the
// next 16 contraction elements and requests a part of a later stage behind each
// product, with addresses that take one addition a stage.  The barrier between two
// stages stands before the products of the last 16 elements of the older one, whose
// fragments are in registers by then; its memory is requested anew from there on (the
// last stages once more where there are none left, so that every step is alike).
struct HeadNoBegin {
  __device__ __forceinline__ void operator()(const HeadSpan&, int) const {}
};
template <class S, bool AROWS, bool BROWS, typename Span, typename Done, typename Begin = HeadNoBegin>
__device__ __forceinline__ void head_product(const HeadProduct& pr, int spans, int total, Span span, Done done,
                                             Begin begin = Begin()) {
  constexpr int kStep = S::kStep;
  typedef typename S::E E;
  typedef HeadType<E> Type;
  using TA = HeadTile<E, S::TM, S::kThreads, AROWS>;
  using TB = HeadTile<E, S::TN, S::kThreads, BROWS>;
  constexpr int kLoads = TA::kLoads + TB::kLoads, KS = 4, MT = S::MT, NT = S::NT;
  static_assert(KS % 2 == 0, "two sets of fragments in turn");
  __shared__ __align__(16384) char sa[S::NS][TA::kBytes];
  __shared__ __align__(16384) char sb[S::NS][TB::kBytes];
  const int tid = threadIdx.x, lane = tid & 63;
  const int w = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int wm = (w % S::WM) * MT * 32, wn = (w / S::WM) * NT * 32;
  const int ksteps = (pr.K + kStep - 1) / kStep;
  const uint32_t at_a = lds_addr_uniform(sa), at_b = lds_addr_uniform(sb);
  const uint32_t la = at_a + TA::template lane_at<true>(wm, lane), lb = at_b + TB::template lane_at<false>(wn, lane);
  // the next request: span, step of it, plane pair, place
  TA ta;
  TB tb;
  int ri = 0, asked = 0, rq, rp, pair_left, rst = 0;
  uint32_t ra = at_a + 1024 * w, rb = at_b + 1024 * w;
  HeadSpan rs;
  auto aim = [&](int k) {
    int x, y;
    head_pair(pr.pa, pr.pb, rp, x, y);
    ta.aim(pr.a, rs.m * S::TM, x, k, tid);
    tb.aim(pr.b, rs.n * S::TN, y, k, tid);
  };
  auto start = [&]() {
    rs = span(ri);
    rq = rs.q0, rp = rq / ksteps;
    const int k = rq - rp * ksteps;
    pair_left = ksteps - k;
    aim(k * kStep);
  };
  start();
  auto request_next = [&]() {   // behind the requests of a stage
    rst = rst + 1 == S::NS ? 0 : rst + 1;
    ra = at_a + 1024 * w + rst * TA::kBytes;
    rb = at_b + 1024 * w + rst * TB::kBytes;
    if (++asked >= total) return;
    ++rq;
    if (rq == rs.q1) {
      ++ri;
      start();
    } else if (--pair_left == 0) {
      ++rp;
      pair_left = ksteps;
      aim(0);
    } else {
      ta.next(pr.a, tid);
      tb.next(pr.b, tid);
    }
  };
  // requests lo .. hi - 1 of a stage
  auto request = [&](auto lo_, auto hi_) {
    head_range<decltype(lo_)::value, decltype(hi_)::value>([&](auto d_) {
      constexpr int d = decltype(d_)::value;
      if constexpr (d < TA::kLoads)
        ta.template request<d>(ra);
      else
        tb.template request<d - TA::kLoads>(rb);
    });
  };
  typename Type::Frag fa[2][MT], fb[2][NT];
  f32x16 acc[MT][NT];
  uint32_t sla = la, slb = lb;   // the stage being read
  // Substep C's products, one pair of fragments a slot; behind them the fragments of substep R are read
  // and the share of a stage's requests that slots S0 .. of kDmaSlots have is made.
  constexpr int kSlots = MT * NT, kReadSlots = kSlots > 4 ? kSlots * 3 / 4 : kSlots;
  constexpr int kDmaSlots = kSlots * (S::NS == 2 ? KS - 1 : KS);
  auto substep = [&](auto c_, auto r_, auto s0_) {
    constexpr int C = decltype(c_)::value, R = decltype(r_)::value, S0 = decltype(s0_)::value;
    head_range<0, kSlots>([&](auto n_) {
      constexpr int n = decltype(n_)::value, i = n / NT, j = n % NT;
      acc[i][j] = Type::product(fa[C & 1][i], fb[C & 1][j], acc[i][j]);
      if constexpr (n < kReadSlots) {
        constexpr int lo = (MT + NT) * n / kReadSlots, hi = (MT + NT) * (n + 1) / kReadSlots;
#pragma unroll
        for (int f = lo; f < hi; ++f) {
          if (f < MT)
            fa[R & 1][f] = TA::frag(sla, f, R);
          else
            fb[R & 1][f - MT] = TB::frag(slb, f - MT, R);
        }
      }
      if constexpr (S0 + n < kDmaSlots)
        request(std::integral_constant<int, kLoads*(S0 + n) / kDmaSlots>{},
                std::integral_constant<int, kLoads*(S0 + n + 1) / kDmaSlots>{});
      __builtin_amdgcn_sched_barrier(0);
    });
  };
  auto clear = [&]() {   // (a product of zeros writes 16 registers in the time of eight moves)
    bf16x8 none = {0, 0, 0, 0, 0, 0, 0, 0};
    const f32x16 zero = {0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0};
#pragma unroll
    for (int i = 0; i < MT; ++i)
#pragma unroll
      for (int j = 0; j < NT; ++j) {
        asm volatile("" : "+v"(none));
        acc[i][j] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(none, none, zero, 0, 0, 0);
      }
  };
  auto arrive = [&]() {   // everybody's part of the next stage, behind which NS - 2 are under way
    vm_wait<(S::NS - 2) * kLoads>();
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");   // (this wave has read the stage before)
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
  };
  constexpr std::integral_constant<int, 0> zero;
  constexpr std::integral_constant<int, kLoads> all;
  constexpr std::integral_constant<int, kLoads * kSlots / kDmaSlots> begun;   // requests made in the last substep
#pragma unroll 1
  for (int i = 0; i < S::NS - 1; ++i) {
    request(zero, all);
    request_next();
  }
  arrive();
#pragma unroll
  for (int i = 0; i < MT; ++i) fa[0][i] = TA::frag(sla, i, 0);
#pragma unroll
  for (int j = 0; j < NT; ++j) fb[0][j] = TB::frag(slb, j, 0);
  request(zero, begun);
  int st = 0;
#pragma unroll 1
  for (int sp = 0; sp < spans; ++sp) {
    const HeadSpan cur = span(sp);
    begin(cur, wn);
    clear();
#pragma unroll 1
    for (int left = cur.q1 - cur.q0; left > 0; --left) {
      head_range<0, KS - 1>([&](auto k_) {
        constexpr int k = decltype(k_)::value;
        substep(k_, std::integral_constant<int, k + 1>{}, std::integral_constant<int, kSlots*(k + 1)>{});
      });
      request_next();
      arrive();
      st = st + 1 == S::NS ? 0 : st + 1;
      sla = la + st * TA::kBytes;
      slb = lb + st * TB::kBytes;
      substep(std::integral_constant<int, KS - 1>{}, zero, zero);
    }
    done(cur, wm, wn, acc);
  }
  vm_wait<0>();   // (nothing arrives in LDS that is another's by then)
}

// Workgroup -> (tile of x's rows, one of `split` lanes over the vocabulary's tiles).
// Workgroups go round-robin over the 8 XCDs: neighbours on one XCD share a tile of
// rows and walk adjacent vocabulary tiles, so that its L2 serves most of both.
struct HeadGrid {
  int n_tiles, split, m_tiles;
};
__device__ __forceinline__ bool head_place(const HeadGrid& g, int bid, int& n, int& lane) {
  if (g.n_tiles >= 8) {
    const int xcd = bid & 7, slot = bid >> 3;
    n = (slot / g.split) * 8 + xcd;
    lane = slot % g.split;
  } else {
    n = bid % g.n_tiles;
    lane = bid / g.n_tiles;
  }
  return n < g.n_tiles;
}

// tiles of vocabulary lane `part` (at least one: split <= m_tiles)
__device__ __forceinline__ int head_share(const HeadGrid& g, int part) {
  return (g.m_tiles - part + g.split - 1) / g.split;
}

__device__ __forceinline__ bool head_real(const int64_t* target, int64_t n, int V) {
  return target != nullptr && target[n] >= 0 && target[n] < V;
}
// What a row's weights refer to: 2^((z - a) log2 e - b), from a maximum m that is one of the
// row's logits.  Near zero a = 0 and b = m log2 e, so that a weight is one multiply-add and an
// exponential; the rounding of b (half a step of it, at most 2^-12) is in every weight alike.
// Far off zero that rounding would be any power of two: there a = m, b = 0.  m starts at the
// lowest finite value, never at a sentinel that a finite logit can lie below.
constexpr float kHeadFar = 4096.0f;
constexpr float kHeadLowest = -3.402823466e38f;
__device__ __forceinline__ bool head_far(float m) { return !(fabsf(m) < kHeadFar); }
struct HeadRef {
  float a, b;
  __device__ __forceinline__ explicit HeadRef(float m) : a(head_far(m) ? m : 0.0f), b(head_far(m) ? 0.0f : m * kLog2e) {}
  __device__ __forceinline__ float weight(float z) const { return fast_exp2(fmaf(z - a, kLog2e, -b)); }
  // what a sum of such weights is multiplied with to refer to `to`
  __device__ __forceinline__ float factor(const HeadRef& to) const {
    return fast_exp2(fmaf(a - to.a, kLog2e, b - to.b));
  }
};

struct HeadFwd {
  HeadProduct pr;    // a: weights, b: rows
  HeadGrid g;
  float2* part;      // [split][N]: maximum and sum of the weights that refer to it
  const int64_t* target;   // or null
  float* zt;         // [N]: the target's z, where there is one
  int N, V;
};

// Log sums over this workgroup's share of the vocabulary.  A lane holds one row of
// x for each of its NT tiles and 16 MT logits of it at a time.
template <class S>
__global__ __launch_bounds__(S::kThreads, S::kPerSimd) void k_head_fwd(const HeadFwd a) {
  int nt, part;
  if (!head_place(a.g, (int)blockIdx.x, nt, part)) return;
  const int lane = threadIdx.x & 63, h = lane >> 5;
  float m[S::NT], l[S::NT];
#pragma unroll
  for (int j = 0; j < S::NT; ++j) m[j] = kHeadLowest, l[j] = 0.0f;
  int t[S::NT];   // the rows' targets
#pragma unroll
  for (int j = 0; j < S::NT; ++j) {
    const int n = nt * S::TN + ((int)threadIdx.x >> 6) / S::WM * S::NT * 32 + 32 * j + (lane & 31);
    t[j] = a.target != nullptr && n < a.N && head_real(a.target, n, a.V) ? (int)a.target[n] : -1;
  }
  const int steps = head_steps<S>(a.pr), tiles = head_share(a.g, part);
  head_product<S, true, true>(
      a.pr, tiles, tiles * steps, [&](int i) { return HeadSpan{part + i * a.g.split, nt, 0, steps}; },
      [&](const HeadSpan& sp, int wm, int wn, f32x16(&acc)[S::MT][S::NT]) {
        const int left = a.V - (sp.m * S::TM + wm + 8 * h);   // tokens from the lane's first one on
        auto add = [&](auto inside) {
#pragma unroll
          for (int j = 0; j < S::NT; ++j) {
            auto z = [&](int i, int r) {   // past the vocabulary: no weight
              return decltype(inside)::value || 32 * i + acc_elem(0, r) < left ? acc[i][j][r] : -__builtin_inff();
            };
            auto sum = [&](float ref) {
              float s[2] = {0.0f, 0.0f};
#pragma unroll
              for (int i = 0; i < S::MT; ++i)
#pragma unroll
                for (int r = 0; r < 16; ++r) s[r & 1] += fast_exp2(fmaf(z(i, r), kLog2e, -ref));
              return s[0] + s[1];
            };
            // the maximum so far serves while no weight has grown past 8 bits (its exponent is rounded
            // to 2^-22 then; a longer way from the maximum would cost the sum digits); the first tile, a
            // row that grows further, one far off zero and one with NaN take their own
            float s = sum(head_far(m[j]) ? __builtin_nanf("") : m[j] * kLog2e);
            if (__any(!(s < 0x1p8f))) {
              float t = z(0, 0);
#pragma unroll
              for (int i = 0; i < S::MT; ++i)
#pragma unroll
                for (int r = 0; r < 16; ++r) t = fmaxf(t, z(i, r));
              const float mn = fmaxf(m[j], t);
              const HeadRef to(mn);
              float own[2] = {0.0f, 0.0f};
#pragma unroll
              for (int i = 0; i < S::MT; ++i)
#pragma unroll
                for (int r = 0; r < 16; ++r) own[r & 1] += to.weight(z(i, r));
              s = own[0] + own[1];
              l[j] *= HeadRef(m[j]).factor(to);
              m[j] = mn;
            }
            l[j] += s;
            // the target's own z: logp is its difference from the sum of the same numbers
            const int at = t[j] - (a.V - left);
            const bool mine = t[j] >= 0 && at >= 0 && at < 32 * S::MT && (at & 8) == 0;
            if (__any(mine)) {
              float zt = 0.0f;
#pragma unroll
              for (int i = 0; i < S::MT; ++i)
#pragma unroll
                for (int r = 0; r < 16; ++r) zt = at == 32 * i + acc_elem(0, r) ? acc[i][j][r] : zt;
              if (mine) a.zt[nt * S::TN + wn + 32 * j + (lane & 31)] = zt;
            }
            __builtin_amdgcn_sched_barrier(0);   // (one row's values in registers at a time)
          }
        };
        if (sp.m * S::TM + S::TM <= a.V)
          add(std::true_type{});
        else
          add(std::false_type{});
      });
  // the halves of a wave, then the waves along the vocabulary
  __shared__ float2 st[S::WM][S::TN];
  const int w = threadIdx.x >> 6, wmi = w % S::WM, wn = (w / S::WM) * S::NT * 32;
#pragma unroll
  for (int j = 0; j < S::NT; ++j) {
    const float mo = __shfl_xor(m[j], 32, kWave), lo = __shfl_xor(l[j], 32, kWave);
    const float mx = fmaxf(m[j], mo);
    const HeadRef to(mx);
    const float s = l[j] * HeadRef(m[j]).factor(to) + lo * HeadRef(mo).factor(to);
    if (h == 0) st[wmi][wn + 32 * j + (lane & 31)] = make_float2(mx, s);
  }
  __syncthreads();
  for (int c = threadIdx.x; c < S::TN; c += S::kThreads) {
    const int n = nt * S::TN + c;
    float mx = kHeadLowest, s = 0.0f;
#pragma unroll
    for (int i = 0; i < S::WM; ++i) mx = fmaxf(mx, st[i][c].x);
    const HeadRef to(mx);
#pragma unroll
    for (int i = 0; i < S::WM; ++i) s += st[i][c].y * HeadRef(st[i][c].x).factor(to);
    if (n < a.N) a.part[(int64_t)part * a.N + n] = make_float2(mx, s);
  }
}

// Joins the shares of a row: a wave a row.
struct HeadJoin {
  const float2* part;
  const float* zt;
  const int64_t* target;   // or null
  float *logp, *lse;
  int64_t N;
  int split, V;
};
__global__ __launch_bounds__(256) void k_head_join(const HeadJoin a) {
  const int lane = threadIdx.x & 63;
  const int64_t n = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
  if (n >= a.N) return;
  const bool real = head_real(a.target, n, a.V);
  const float zt = a.zt[n];   // (asked for here, not behind the sums; of no meaning where there is no target)
  float m = kHeadLowest, l = 0.0f;
  constexpr int kAtOnce = 4;
  for (int s0 = 0; s0 < a.split; s0 += kAtOnce * kWave) {
    float2 p[kAtOnce];
    float mx = m;
#pragma unroll
    for (int u = 0; u < kAtOnce; ++u) {
      const int s = s0 + u * kWave + lane;
      p[u] = s < a.split ? a.part[(int64_t)s * a.N + n] : make_float2(kHeadLowest, 0.0f);
    }
#pragma unroll
    for (int u = 0; u < kAtOnce; ++u) mx = fmaxf(mx, p[u].x);
    mx = wave_max(mx);
    const HeadRef to(mx);
    l *= HeadRef(m).factor(to);
#pragma unroll
    for (int u = 0; u < kAtOnce; ++u) l += p[u].y * HeadRef(p[u].x).factor(to);
    m = mx;
  }
  const HeadRef ref(m);
  const bool nan = l != l;   // (a maximum passes NaN over: its sum shows it)
  l = wave_sum(l);
  if (__any(nan) || l == 0.0f) l = __builtin_nanf("");   // (no weight at all: every logit is minus infinity)
  if (lane != 0) return;
  // l = f 2^e with f about 1.  The target's distance from the maximum and e are joined in 64
  // bits, so that logp is off by a few 2^-24 however large the logits are (less lse it would
  // have an error of lse's size: 8e-6 at 100, of either sign).
  int e;
  float f = frexpf(l, &e);
  if (f < 0.70710678f) f *= 2.0f, --e;
  const float log_f = __log2f(f);
  constexpr double kPerBit = 1.0 / (double)kLog2e;
  a.lse[n] = (float)((double)ref.a + ((double)ref.b + (double)e + (double)log_f) * kPerBit);
  if (a.target == nullptr) return;
  float logp = 0.0f;
  if (real) {
    const double d = fma((double)zt - (double)ref.a, (double)kLog2e, -(double)ref.b) - (double)e;
    logp = ((float)d - log_f) * (float)kPerBit;
    logp = logp > 0.0f ? 0.0f : logp;   // (NaN stays)
  }
  a.logp[n] = logp;
}

// dz of a piece of the vocabulary, as the gradients' operand
struct HeadDz {
  HeadProduct pr;
  HeadGrid g;
  const float *lse, *dlogp, *dlse;   // dlogp, dlse: or null
  const int64_t* target;             // or null
  void* dz;                          // [planes][N rounded up to 64][ld], zeros past N and past the vocabulary
  int64_t ld, plane;
  int N, V, v0;                      // the piece starts at token v0 (V: of the whole vocabulary)
  int vocab;                         // ... and has so many
  int rows;                          // N rounded up to 64
};
// The bf16 plane of v that comes next; v becomes what it leaves.  neg: a sign bit to flip.
__device__ __forceinline__ u32x4 next_plane(float (&v)[8], uint32_t neg) {
  bf16x8 o;
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    o[j] = (bf16)v[j];
    v[j] -= (float)o[j];
  }
  return __builtin_bit_cast(u32x4, o) ^ (neg | neg >> 16);
}
template <class S, int PLANES>
__global__ __launch_bounds__(S::kThreads, S::kPerSimd) void k_head_dz(const HeadDz a) {
  int nt, part;
  if (!head_place(a.g, (int)blockIdx.x, nt, part)) return;
  const int lane = threadIdx.x & 63, h = lane >> 5;
  const int wn0 = ((threadIdx.x >> 6) / S::WM) * S::NT * 32;
  float off[S::NT];      // |dz| = 2^(z log2 e - off), of a row far off zero with z - lse (<= 0) for z
  uint32_t neg[S::NT];   // dz's sign bit
  bool far = false;
#pragma unroll
  for (int j = 0; j < S::NT; ++j) {
    const int n = nt * S::TN + wn0 + 32 * j + (lane & 31);
    off[j] = __builtin_inff();   // (nothing weighs anything)
    neg[j] = 0;
    if (n < a.N) {
      float co = a.dlse != nullptr ? a.dlse[n] : 0.0f;
      if (a.dlogp != nullptr && head_real(a.target, n, a.V)) co -= a.dlogp[n];
      const float lse = a.lse[n];
      far = far || head_far(lse);
      // (lse - lse: NaN stays NaN)
      if (co != 0.0f) off[j] = (head_far(lse) ? lse - lse : lse * kLog2e) - __log2f(fabsf(co));
      neg[j] = __float_as_uint(co) & 0x80000000u;
    }
  }
  // Results turn in LDS, 32 tokens x 128 bytes of the vocabulary a wave at a time, so that eight
  // lanes store 128 bytes in a row: a store of 32 rows takes the caches four times as many requests.
  typedef typename S::E E;
  constexpr int kC = 16 / (int)sizeof(E), kI = 4 / (int)sizeof(E);   // elements of 16 bytes; 32-row tiles of 128
  static_assert(S::MT % kI == 0 && (kI == 2 || PLANES == 1), "128 bytes of the vocabulary");
  __shared__ __align__(16) char turn[S::kThreads / 64 * 4096];
  const int steps = head_steps<S>(a.pr), tiles = head_share(a.g, part);
  const bool any_far = __any(far) != 0;
  head_product<S, true, true>(
      a.pr, tiles, tiles * steps, [&](int i) { return HeadSpan{part + i * a.g.split, nt, 0, steps}; },
      [&](const HeadSpan& sp, int wm, int wn, f32x16(&acc)[S::MT][S::NT]) {
        const int mt = sp.m;
        if (any_far) {
#pragma unroll
          for (int j = 0; j < S::NT; ++j) {
            const int n = nt * S::TN + wn + 32 * j + (lane & 31);
            const float lse = n < a.N ? a.lse[n] : 0.0f;
            const float from = head_far(lse) ? lse : 0.0f, most = head_far(lse) ? 0.0f : __builtin_inff();
#pragma unroll
            for (int i = 0; i < S::MT; ++i)
#pragma unroll
              for (int r = 0; r < 16; ++r)   // (a row without weight has no gradient, whatever its logits)
                acc[i][j][r] = off[j] == __builtin_inff() ? 0.0f : fminf(acc[i][j][r] - from, most);
          }
        }
        // else zeros past the vocabulary, and in the rows past N (of any sums, NaN among them)
        const bool inside = mt * S::TM + S::TM <= a.vocab && nt * S::TN + S::TN <= a.N;
        char* const mine = turn + (threadIdx.x >> 6) * 4096;
        char* const put = mine + (lane & 31) * 128;
        const int put_key = (lane >> 1) & 7;
        const int v0 = mt * S::TM + wm, n0 = nt * S::TN + wn;
#pragma unroll
        for (int j = 0; j < S::NT; ++j) {
          const bool real = n0 + 32 * j + (lane & 31) < a.N;
#pragma unroll
          for (int i = 0; i < S::MT; i += kI) {
            float d[2 * kI][8];
#pragma unroll
            for (int q = 0; q < PLANES; ++q) {
#pragma unroll
              for (int c = 0; c < 2 * kI; ++c) {   // 8 elements from v0 + 32 i + 16 c + 8 h on
                if (q == 0) {
#pragma unroll
                  for (int r = 0; r < 8; ++r)
                    d[c][r] = fast_exp2(fmaf(acc[i + c / 2][j][8 * (c % 2) + r], kLog2e, -off[j]));
                  if (!inside) {
#pragma unroll
                    for (int r = 0; r < 8; ++r)
                      if (v0 + 32 * i + 16 * c + 8 * h + r >= a.vocab || !real) d[c][r] = 0.0f;
                  }
                }
                if constexpr (kC == 8) {
                  *reinterpret_cast<u32x4*>(put + (((2 * c + h) ^ put_key) << 4)) = next_plane(d[c], neg[j]);
                } else {
#pragma unroll
                  for (int x = 0; x < 2; ++x) {
                    const f32x4 o = {d[c][4 * x], d[c][4 * x + 1], d[c][4 * x + 2], d[c][4 * x + 3]};
                    *reinterpret_cast<u32x4*>(put + (((4 * c + 2 * h + x) ^ put_key) << 4)) =
                        __builtin_bit_cast(u32x4, o) ^ neg[j];
                  }
                }
                __builtin_amdgcn_sched_barrier(0);
              }
              // (a wave's LDS requests are served in order: the compiler alone has to keep it)
              asm volatile("" ::: "memory");
              __builtin_amdgcn_wave_barrier();
#pragma unroll
              for (int t = 0; t < 4; ++t) {
                const int r = 8 * t + (lane >> 3), n = n0 + 32 * j + r;
                const u32x4 o = *reinterpret_cast<const u32x4*>(mine + r * 128 + (((lane & 7) ^ ((r >> 1) & 7)) << 4));
                if (n < a.rows)
                  *reinterpret_cast<u32x4*>(static_cast<E*>(a.dz) + q * a.plane + (int64_t)n * a.ld + v0 + 32 * i +
                                            kC * (lane & 7)) = o;
              }
              asm volatile("" ::: "memory");
              __builtin_amdgcn_wave_barrier();
            }
          }
        }
      });
}

// The target's own element, a p_t + b, of a row that has one.
__device__ __forceinline__ float head_target(float b, float dl, float lp) {
  if (b == 0.0f && dl == 0.0f) return 0.0f;   // (whatever the row's logits)
  // (dlse - b) p + b with 1 - p from expm1: within a few 2^-24 as logp is, not of the size of the logits
  return dl * expf(lp) - b * expm1f(lp);
}
__device__ __forceinline__ float head_target(const HeadDz& a, const float* logp, int64_t n) {
  return head_target(a.dlogp[n], a.dlse != nullptr ? a.dlse[n] : 0.0f, logp[n]);
}
// ... where the piece has it, and (rest: not null) what its rounding to bf16 leaves of it with
// its token; 0 and -1 without one.
template <typename E, int PLANES>
__global__ __launch_bounds__(256) void k_head_target(const HeadDz a, const float* logp, float* rest, int* token) {
  const int64_t n = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (n >= a.N || a.dlogp == nullptr) return;
  const bool real = head_real(a.target, n, a.V);
  const int64_t t = real ? a.target[n] : -1, v = t - a.v0;
  float d = real ? head_target(a, logp, n) : 0.0f;
  if (rest != nullptr) {
    rest[n] = d - (float)(bf16)d;
    token[n] = (int)t;
  }
  if (!real || v < 0 || v >= a.vocab) return;
  E* p = static_cast<E*>(a.dz) + n * a.ld + v;
#pragma unroll
  for (int q = 0; q < PLANES; ++q) {
    const E o = (E)d;
    p[q * a.plane] = o;
    d -= (float)o;
  }
}

// Both for up to 2048 rows of x, and the rests' sums by token, in one launch.  More rows are
// sorted by token (2048 rows of 768: 22 us, 29 sorted; 4096: 45 and 38).  A workgroup takes 16
// rows, each by a wave; the first row of a token sums them all, a wave those of a token of few
// rows, the workgroup those of one of many.  sums[n] where n is such a row; first[t_n] = n, and
// other tokens' `first` is left as it was: `there` has the tokens' bits, 65536 of them a workgroup.
constexpr int kFewRows = 2048, kFewThreads = 1024, kFewWaves = kFewThreads / 64, kFewAlone = 8;
constexpr int kFewBits = 1 << 16;
struct HeadFewRows {
  HeadDz z;
  const float* logp;
  const bf16* x;
  float* rest;
  int* token;
  bf16* sums;          // null: no sums
  int* first;
  uint64_t* there;     // [V rounded up to 256, / 64]
  int D;
};
__global__ __launch_bounds__(kFewThreads) void k_head_few(const HeadFewRows a) {
  constexpr int kPer = kFewRows / kFewThreads, kWords = kFewRows / 64;
  __shared__ int token[kFewRows];
  __shared__ float weight[kFewRows];
  __shared__ uint64_t same[kFewWaves][kWords];   // of the wave's row: the rows of its token, 64 a word
  __shared__ int count[kFewWaves];               // ... how many, 0 but for its first
  __shared__ float part[kFewWaves][512];
  unsigned* const bits = reinterpret_cast<unsigned*>(part);
  static_assert(sizeof(part) >= kFewBits / 8, "a workgroup's bits");
  const int tid = threadIdx.x, lane = tid & 63, w = tid >> 6, N = a.z.N, D = a.D;
  const int words = (N + 63) / 64, n = (int)blockIdx.x * kFewWaves + w;
  // all that one waits for at once: the rows' numbers, and the wave's own row of x
  constexpr int kOwn = 2;
  bf16x8u own[kOwn];
#pragma unroll
  for (int u = 0; u < kOwn; ++u) {
    const int c = 8 * (64 * u + lane);
    if (n < N && c + 8 <= D) own[u] = *reinterpret_cast<const bf16x8u*>(a.x + (int64_t)n * D + c);
  }
  int64_t t[kPer];
  float b[kPer], dl[kPer], lp[kPer];
#pragma unroll
  for (int u = 0; u < kPer; ++u) {
    const int i = u * kFewThreads + tid;
    t[u] = i < N ? a.z.target[i] : -1;
    b[u] = i < N ? a.z.dlogp[i] : 0.0f;
    dl[u] = i < N && a.z.dlse != nullptr ? a.z.dlse[i] : 0.0f;
    lp[u] = i < N ? a.logp[i] : 0.0f;
  }
  const int64_t bit0 = (int64_t)blockIdx.x * kFewBits;
  const bool has_bits = bit0 < a.z.V;
  if (has_bits)
    for (int i = tid; i < kFewBits / 32; i += kFewThreads) bits[i] = 0;
#pragma unroll
  for (int u = 0; u < kPer; ++u) {
    const int i = u * kFewThreads + tid;
    if (u * kFewThreads >= N) break;
    const bool real = t[u] >= 0 && t[u] < a.z.V;
    const float d = real ? head_target(b[u], dl[u], lp[u]) : 0.0f;
    const bf16 o = (bf16)d;
    token[i] = real ? (int)t[u] : -1;
    weight[i] = d - (float)o;
    if (i < N && i / kFewWaves == (int)blockIdx.x) {
      a.rest[i] = d - (float)o;
      a.token[i] = real ? (int)t[u] : -1;
      const int64_t v = t[u] - a.z.v0;
      if (real && v >= 0 && v < a.z.vocab) static_cast<bf16*>(a.z.dz)[i * a.z.ld + v] = o;
    }
  }
  if (a.sums == nullptr) return;
  __syncthreads();
  if (has_bits) {   // the tokens that are there, of this workgroup's
    for (int i = tid; i < N; i += kFewThreads) {
      const int64_t v = token[i] - bit0;
      if (token[i] >= 0 && v >= 0 && v < kFewBits) atomicOr(&bits[v / 32], 1u << (v & 31));
    }
  }
  const int mine = n < N ? token[n] : -1;
  int found = 0;
  if (mine >= 0) {   // (uniform over the wave)
    bool before = false;
#pragma unroll 8
    for (int k = 0; k < words; ++k) {
      const uint64_t m = __ballot(64 * k + lane < N && token[64 * k + lane] == mine);
      before = before || (64 * k + 63 < n ? m : 64 * k > n ? 0 : m & ((1ull << (n & 63)) - 1ull)) != 0;
      found += __popcll(m);
      if (lane == 0) same[w][k] = m;
    }
    if (before) found = 0;
    if (lane == 0 && found > 0) a.first[mine] = n;
  }
  if (lane == 0) count[w] = found;
  __syncthreads();
  if (has_bits) {
    const int64_t all = ((int64_t)a.z.V + 255) / 256 * 4, at = bit0 / 64;
    for (int i = tid; i < kFewBits / 64 && at + i < all; i += kFewThreads)
      a.there[at + i] = (uint64_t)bits[2 * i + 1] << 32 | bits[2 * i];
  }
  // the rows of `m` (rows 64 k ..), in order, 8 columns a lane from c on
  auto add = [&](float(&acc)[8], uint64_t m, int k, int c) {
    while (m != 0) {
      float v[4][8], f[4];
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        const int r = 64 * k + (m != 0 ? __builtin_ctzll(m) : 0);
        f[u] = m != 0 ? weight[r] : 0.0f;
        load_run8(a.x + (int64_t)r * D + c, m != 0 ? D - c : 0, v[u]);
        m &= m - 1;
      }
#pragma unroll
      for (int u = 0; u < 4; ++u)
#pragma unroll
        for (int j = 0; j < 8; ++j) acc[j] = fmaf(f[u], v[u][j], acc[j]);
    }
  };
  if (found == 1) {
    const float f = weight[n];
    auto store = [&](int c, float(&v)[8]) {
#pragma unroll
      for (int j = 0; j < 8; ++j) v[j] *= f;
      store_run8(a.sums + (int64_t)n * D + c, D - c, v);
    };
#pragma unroll
    for (int u = 0; u < kOwn; ++u) {
      const int c = 8 * (64 * u + lane);
      if (c >= D) continue;
      float v[8];
      if (c + 8 <= D) {
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] = (float)own[u][j];
      } else {
        load_run8(a.x + (int64_t)n * D + c, D - c, v);
      }
      store(c, v);
    }
#pragma unroll 4
    for (int c = 8 * (64 * kOwn + lane); c < D; c += 512) {
      float v[8];
      load_run8(a.x + (int64_t)n * D + c, D - c, v);
      store(c, v);
    }
  } else if (found > 0 && found <= kFewAlone) {
    for (int c = 8 * lane; c < D; c += 512) {
      float acc[8] = {0, 0, 0, 0, 0, 0, 0, 0};
      for (int k = n / 64; k < words; ++k) add(acc, same[w][k], k, c);
      store_run8(a.sums + (int64_t)n * D + c, D - c, acc);
    }
  }
  uint64_t many = __ballot(lane < kFewWaves && count[lane & (kFewWaves - 1)] > kFewAlone);   // (every wave: the same)
  while (many != 0) {
    const int q = __builtin_ctzll(many);
    many &= many - 1;
    const int64_t row = (int64_t)blockIdx.x * kFewWaves + q;
    for (int c0 = 0; c0 < D; c0 += 512) {
      float acc[8] = {0, 0, 0, 0, 0, 0, 0, 0};
      if (c0 + 8 * lane < D)
        for (int k = w; k < words; k += kFewWaves) add(acc, same[q][k], k, c0 + 8 * lane);
      __syncthreads();   // (`part` is read no more)
#pragma unroll
      for (int j = 0; j < 8; ++j) part[w][8 * lane + j] = acc[j];
      __syncthreads();
      const int c = c0 + tid;
      if (tid < 512 && c < D) {
        float t = 0.0f;
        for (int k = 0; k < kFewWaves; ++k) t += part[k][tid];
        a.sums[row * D + c] = (bf16)t;
      }
    }
  }
}

// Rows of bf16 that go to the results' rows beside the products: W_{t_n} with the weight
// rest_n to row n of dx, the sum of a token's rest_n x_n (rounded to bf16: of a part that is
// 2^-8 of the whole) to its row of dW.
struct HeadMore {
  const bf16* rows;          // null: none
  int64_t ld;
  const int* token;          // dx: of every row, or -1
  const float* weight;
  const int* first;          // dW: a token's row,
  const uint64_t* there;     // ... of the tokens that have one: a bit each
};
// The bits of 32 tokens from n0 (the same in a wave) on, by a scalar load: a vector load would wait for the product's
// requests ahead of it, also where no token has a row.
__device__ __forceinline__ uint32_t head_there(const HeadMore& a, int64_t n0) {
  typedef const __attribute__((address_space(4))) uint32_t* Words;
  return ((Words)(uintptr_t)a.there)[__builtin_amdgcn_readfirstlane((int)(n0 / 32))];
}

// dx (rows of x on n, columns of W on m) and dW (tokens on n, columns of x on m).  The
// workgroups take whole tiles in rounds, neighbours on one XCD at the same steps, so
// that its L2 serves them all; the tiles of a last round that would not fill the chip
// are cut into `cuts` parts each, which go to `part` and are added by
// k_head_join_tiles.  So do whole tiles that reach past D: their rows' ends are written
// there.
struct HeadGrad {
  HeadProduct pr;
  void* out;             // [N][D]: float32 or, out_bf16, bf16
  const float* add;      // float32 of the same shape to add, or null
  float* part;           // [cuts][tiles - whole][TN][TM], then [n_tiles][TN][TM] of the edge
  int N, D, m_tiles, n_tiles, groups;
  int whole, cuts;       // tiles taken whole, a multiple of groups
  bool out_bf16;
  HeadMore more;
};

template <class S, bool BROWS>
__global__ __launch_bounds__(S::kThreads, S::kPerSimd) void k_head_grad(const HeadGrad a) {
  const int g = (int)xcd_remap(blockIdx.x, gridDim.x);
  const int steps = head_steps<S>(a.pr), rounds = a.whole / a.groups;
  const int rest = a.m_tiles * a.n_tiles - a.whole, units = rest * a.cuts;
  // whole tiles, then units g, g + groups, ..: unit u is part u / rest of tile whole + u % rest
  auto span = [&](int i) {
    int t = i * a.groups + g, q0 = 0, q1 = steps;
    if (i >= rounds) {
      const int u = (i - rounds) * a.groups + g, c = u / rest;
      t = a.whole + u % rest;
      q0 = (int)((int64_t)steps * c / a.cuts);
      q1 = (int)((int64_t)steps * (c + 1) / a.cuts);
    }
    return HeadSpan{t % a.m_tiles, t / a.m_tiles, q0, q1};
  };
  const int spans = rounds + (g < units ? (units - g + a.groups - 1) / a.groups : 0);
  int total = 0;
  for (int i = 0; i < spans; ++i) {
    const HeadSpan sp = span(i);
    total += sp.q1 - sp.q0;
  }
  if (total == 0) return;
  const int lane = threadIdx.x & 63, h = lane >> 5;
  constexpr bool kMore = sizeof(typename S::E) == 2;   // (float32 operands: none)
  // asked for a tile ahead: dx: the rows' tokens and weights; dW: the tokens' bits
  int token[S::NT];
  float weight[S::NT];
  uint32_t there[S::NT];
  const bool more = kMore && a.more.rows != nullptr;
  auto begin = [&](const HeadSpan& sp, int wn) {
    if (!more) return;
#pragma unroll
    for (int j = 0; j < S::NT; ++j) {
      const int64_t n0 = (int64_t)sp.n * S::TN + wn + 32 * j, n = n0 + (lane & 31) < a.N ? n0 + (lane & 31) : a.N - 1;
      if (BROWS) {
        token[j] = a.more.token[n];
        weight[j] = a.more.weight[n];
      } else {
        there[j] = head_there(a.more, n0 < a.N ? n0 : 0);
      }
    }
  };
  head_product<S, false, BROWS>(
      a.pr, spans, total, span, [&](const HeadSpan& sp, int wm, int wn, f32x16(&acc)[S::MT][S::NT]) {
        const int t = sp.n * a.m_tiles + sp.m;
        float* part = nullptr;
        if (sp.q1 - sp.q0 != steps) {   // (cuts <= steps: the part that ends at q1)
          const int c = (int)(((int64_t)sp.q1 * a.cuts + steps - 1) / steps) - 1;
          part = a.part + ((int64_t)c * rest + t - a.whole) * S::TM * S::TN;
        }
        if (part == nullptr && sp.m * S::TM + S::TM > a.D) part = a.part + ((int64_t)units + sp.n) * S::TM * S::TN;
        // a lane's runs of a row: 32 i + 2 r0 elements from its first one on, two tiles' at a time
        constexpr int kAhead = S::MT % 2 == 0 ? 4 : 2;
        auto each = [&](auto to, auto ask, auto put) {
#pragma unroll
          for (int j = 0; j < S::NT; ++j) {
            const int c = wn + 32 * j + (lane & 31);
            if (sp.n * (int64_t)S::TN + c >= a.N) continue;
            const auto at = to(c, wm + 8 * h, j);
#pragma unroll
            for (int k0 = 0; k0 < 2 * S::MT; k0 += kAhead) {
              bf16x8u u[kAhead];
#pragma unroll
              for (int k = 0; k < kAhead; ++k) ask(at, 16 * (k0 + k), u[k]);
              __builtin_amdgcn_sched_barrier(0);
#pragma unroll
              for (int k = 0; k < kAhead; ++k) {
                float v[8];
#pragma unroll
                for (int r = 0; r < 8; ++r) v[r] = acc[(k0 + k) / 2][j][8 * (k & 1) + r];
                put(at, 16 * (k0 + k), u[k], v);
                __builtin_amdgcn_sched_barrier(0);   // (few of the results in other registers at a time)
              }
            }
          }
        };
        struct At {
          int64_t at;
          const bf16* more;
          float weight;
          bool some;   // the wave has any
        };
        auto in_out = [&](int c, int e, int j) {
          At to{((int64_t)sp.n * S::TN + c) * a.D + sp.m * S::TM + e, nullptr, 0.0f, false};
          if (more && (BROWS || there[j] != 0)) {
            to.some = true;
            int row = -1;
            if (BROWS)
              row = token[j];
            else if ((there[j] >> (lane & 31)) & 1u)
              row = a.more.first[(int64_t)sp.n * S::TN + c];
            if (row >= 0) to.more = a.more.rows + row * a.more.ld + sp.m * S::TM + e;
            to.weight = BROWS ? weight[j] : 1.0f;
          }
          return to;
        };
        auto ask = [&](const At& to, int o, bf16x8u& u) {
          if (to.some && to.more != nullptr) u = *reinterpret_cast<const bf16x8u*>(to.more + o);
        };
        auto added = [&](const At& to, int o, const bf16x8u& u, float(&v)[8]) {
          if (a.add != nullptr) {
            float f[8];
            load_run8(a.add + to.at + o, f);
#pragma unroll
            for (int r = 0; r < 8; ++r) v[r] += f[r];
          }
          if (to.some && to.more != nullptr) {
#pragma unroll
            for (int r = 0; r < 8; ++r) v[r] = fmaf(to.weight, (float)u[r], v[r]);
          }
        };
        if (part != nullptr) {
          each([&](int c, int e, int) { return part + c * S::TM + e; }, [](float*, int, bf16x8u&) {},
               [&](float* at, int o, const bf16x8u&, float(&v)[8]) { store_run8(at + o, v); });
        } else if (a.out_bf16) {
          each(in_out, ask, [&](const At& to, int o, const bf16x8u& u, float(&v)[8]) {
            added(to, o, u, v);
            store_run8(static_cast<bf16*>(a.out) + to.at + o, v);
          });
        } else {
          each(in_out, ask, [&](const At& to, int o, const bf16x8u& u, float(&v)[8]) {
            added(to, o, u, v);
            store_run8(static_cast<float*>(a.out) + to.at + o, v);
          });
        }
      },
      begin);
}

// The cut tiles' parts in order, and the tiles at the rows' ends.  Eight workgroups a
// tile, a thread 8 elements at a time.
template <class S, bool DX>
__global__ __launch_bounds__(256) void k_head_join_tiles(const HeadGrad a, int first) {
  const int t = first + (int)blockIdx.x, rest = a.m_tiles * a.n_tiles - a.whole;
  const int m0 = (t % a.m_tiles) * S::TM;
  const bool cut = t >= a.whole && a.cuts > 1;
  if (!cut && m0 + S::TM <= a.D) return;
  const int64_t n0 = (int64_t)(t / a.m_tiles) * S::TN;
  const float* part =
      a.part + (cut ? (int64_t)t - a.whole : (int64_t)rest * a.cuts + t / a.m_tiles) * S::TM * S::TN;
  const int64_t next = (int64_t)rest * S::TM * S::TN;
  constexpr int kRuns = S::TM / 8;
  for (int i = (int)blockIdx.y * 256 + threadIdx.x; i < S::TN * kRuns; i += 8 * 256) {
    const int c = i / kRuns, e = i % kRuns * 8, d = m0 + e;
    const int64_t n = n0 + c;
    if (n >= a.N || d >= a.D) continue;
    float v[8], u[8];
    load_run8(part + c * S::TM + e, v);
#pragma unroll 4
    for (int g = 1; g < (cut ? a.cuts : 1); ++g) {
      load_run8(part + g * next + c * S::TM + e, u);
#pragma unroll
      for (int r = 0; r < 8; ++r) v[r] += u[r];
    }
    if (a.add != nullptr) {
      load_run8(a.add + n * a.D + d, a.D - d, u);
#pragma unroll
      for (int r = 0; r < 8; ++r) v[r] += u[r];
    }
    if (a.more.rows != nullptr) {
      int row = -1;
      if (DX)
        row = a.more.token[n];
      else if ((reinterpret_cast<const uint32_t*>(a.more.there)[n / 32] >> (n & 31)) & 1u)
        row = a.more.first[n];
      if (row >= 0) {
        const float weight = DX ? a.more.weight[n] : 1.0f;
        load_run8(a.more.rows + row * a.more.ld + d, a.D - d, u);
#pragma unroll
        for (int r = 0; r < 8; ++r) v[r] = fmaf(weight, u[r], v[r]);
      }
    }
    if (a.out_bf16)
      store_run8(static_cast<bf16*>(a.out) + n * a.D + d, a.D - d, v);
    else
      store_run8(static_cast<float*>(a.out) + n * a.D + d, a.D - d, v);
  }
}

// Rows as bf16 planes or float32 with a pitch of ld: [planes][rows][ld], zeros past a row.
template <typename E, int PLANES>
__global__ __launch_bounds__(256) void k_head_pack(const void* x, bool x_bf16, E* out, int64_t rows, int D, int ld) {
  const int runs = ld / 8;
  const int64_t total = rows * runs, plane = rows * ld;
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < total; i += (int64_t)gridDim.x * 256) {
    const int64_t r = i / runs;
    const int c = (int)(i % runs) * 8;
    float v[8];
    load_run8_of(x, x_bf16, r * D + c, D - c, v);
    if constexpr (sizeof(E) == 4) {
      store_run8(out + r * ld + c, v);
    } else {
#pragma unroll
      for (int q = 0; q < PLANES; ++q) *reinterpret_cast<u32x4*>(out + q * plane + r * ld + c) = next_plane(v, 0);
    }
  }
}

// ---------------------------------------------------------------------------
// host
// ---------------------------------------------------------------------------
template <typename E> using HeadBig = HeadShape<256, 256, 2, 4, 2, 1, E>;
template <typename E> using HeadMid = HeadShape<128, 128, 2, 2, 2, 2, E>;
template <typename E> using HeadFew = HeadShape<128, 32, 4, 1, 4, 1, E>;
template <typename E> using HeadFew64 = HeadShape<128, 64, 2, 2, 3, 2, E>;
using HeadFewBack = HeadShape<128, 64, 2, 2, 3, 1, float>;   // (the backward's, up to 64 rows)
template <typename E> using HeadFew128 = HeadShape<128, 128, 2, 2, 4, 1, E>;

static bool head_type(int dtype) { return dtype == NSA_F32 || dtype == NSA_BF16; }
static bool head_shape_ok(int64_t N, int V, int D) {
  return N >= 0 && N <= kHeadRows && V >= 1 && V <= kHeadVocab && D >= 1 && D <= kHeadWide;
}
static size_t up16(size_t n) { return (n + 255) / 256 * 256; }

// Tile of the product over the vocabulary: 256 x 256 where that gives five of eight compute
// units a tile (16000 x 768, 700 rows, 0.74 of them: 29.5 us, 33 in 128 x 128; 8192 x 768, 1024 rows,
// 0.5: 28 and 25), else 128 x 128.  The forward of up to 128 rows, one tile across, waits for W: it
// takes the narrowest of 32, 64 and 128 rows, with stages for more of W under way (bf16, W
// 32000 x 4096, 64 and 128 rows: 50 and 53 us, 67 and 71 in the common 128 x 128).
enum { kFew, kFew64, kFew128, kMid, kBig };
static int head_kind(int64_t N, int V, int cu) {
  return ((N + 255) / 256) * ((V + 255) / 256) * 8 >= (int64_t)cu * 5 && N > 128 ? kBig : kMid;
}
static int head_fwd_kind(int64_t N, int V, int cu) {
  return N <= 32 ? kFew : N <= 64 ? kFew64 : N <= 128 ? kFew128 : head_kind(N, V, cu);
}
// Whether float32 rows and weights go through the float32 instructions rather than as
// planes.  Planes take six products of bf16 at 870 to 1150 TFLOP/s together and a copy of
// W of 1.5 times its size, the float32 instructions up to 140 TFLOP/s and no copy: they win
// where rows are few and the tiles of 128 x 128 half fill the chip.  Measured, us of the instructions
// and of planes, in the order of the W's 32000 x 768, 50257 x 1024, 8192 x 4096 and 128000 x 2048:
//   forward   128 rows  59  90   130  210   247 248    498 1010
//             512      186 167   474  380   248 443   1876 1760
//             768      275 241   594  516   468 438   2813 2331
//   backward  128 rows 203 245   378  467   486 493   1587 2275
//             256      309 322   671  646   530 613   2933 2898
//             512      571 539  1251 1020   755 830   5651 4735
static bool head_native(int64_t N, int V, int most, int cu) {
  return N <= 64 || (N <= most && (N + 127) / 128 * ((V + 127) / 128) * 2 >= cu);
}
constexpr int kNativeFwd = 512, kNativeBwd = 256;

// How the operands lie: as given, or packed (planes, padded rows).
struct HeadLayout {
  bool native, pack_x, pack_w;  // native: products of float32
  int px, pw, ld;               // planes; pitch of a packed row
  size_t x_bytes, w_bytes;      // of the packed copies
};
static HeadLayout head_layout(int64_t N, int V, int D, const void* x, const void* w, int x_dtype, int w_dtype, int native, int cu) {
  HeadLayout l;
  const bool wide = x_dtype == NSA_F32, both = wide && w_dtype == NSA_F32;
  l.native = both && head_native(N, V, native, cu);
  l.px = wide && !l.native ? 3 : 1;
  l.pw = both && !l.native ? 3 : 1;
  l.ld = (D + 63) / 64 * 64;
  // rows are requested in whole stages, aligned pieces of 16 bytes
  const int step = l.native ? 32 : 64, size = l.native ? 4 : 2;
  l.pack_x = l.px == 3 || D % step != 0 || reinterpret_cast<uintptr_t>(x) % 16 != 0;
  l.pack_w = (w_dtype == NSA_F32 && !l.native) || D % step != 0 || reinterpret_cast<uintptr_t>(w) % 16 != 0;
  l.x_bytes = l.pack_x ? up16((size_t)l.px * N * l.ld * size) : 0;
  l.w_bytes = l.pack_w ? up16((size_t)l.pw * V * l.ld * size) : 0;
  return l;
}
static void head_pack(const void* x, int dtype, void* out, int64_t rows, int D, int ld, int planes, bool native,
                      hipStream_t s) {
  const int64_t blocks = (rows * (ld / 8) + 255) / 256;
  const unsigned grid = (unsigned)(blocks < 65536 ? blocks : 65536);
  const bool half = dtype == NSA_BF16;
  if (native)
    k_head_pack<float, 1><<<grid, 256, 0, s>>>(x, half, static_cast<float*>(out), rows, D, ld);
  else if (planes == 3)
    k_head_pack<bf16, 3><<<grid, 256, 0, s>>>(x, half, static_cast<bf16*>(out), rows, D, ld);
  else
    k_head_pack<bf16, 1><<<grid, 256, 0, s>>>(x, half, static_cast<bf16*>(out), rows, D, ld);
}

template <class S>
static HeadGrid head_grid(int64_t N, int vocab, int cu) {
  HeadGrid g;
  g.n_tiles = (int)((N + S::TN - 1) / S::TN);
  g.m_tiles = (vocab + S::TM - 1) / S::TM;
  // rounds of the chip's workgroups, a workgroup's tiles and half a tile to begin and end
  const int64_t at_once = (int64_t)cu * S::kPerCu;
  double best = 1e30;
  g.split = 1;
  for (int s = 1; s <= g.m_tiles && (s == 1 || (int64_t)s * g.n_tiles <= 4 * at_once); ++s) {
    const double time = (double)((s * (int64_t)g.n_tiles + at_once - 1) / at_once) * ((g.m_tiles + s - 1) / s + 0.5);
    if (time < best) best = time, g.split = s;
  }
  return g;
}
static unsigned head_blocks(const HeadGrid& g) {
  return (unsigned)((g.n_tiles >= 8 ? (g.n_tiles + 7) / 8 * 8 : g.n_tiles) * (int64_t)g.split);
}
// f with the shape of the forward's tiles
template <typename F>
static auto head_as(int kind, bool native, F f) {
  if (native)
    return kind == kFew     ? f(HeadFew<float>{})
           : kind == kFew64 ? f(HeadFew64<float>{})
           : kind == kFew128 ? f(HeadFew128<float>{})
                             : f(HeadMid<float>{});
  return kind == kFew     ? f(HeadFew<bf16>{})
         : kind == kFew64 ? f(HeadFew64<bf16>{})
         : kind == kFew128 ? f(HeadFew128<bf16>{})
         : kind == kMid    ? f(HeadMid<bf16>{})
                           : f(HeadBig<bf16>{});
}

// The gradients' products: tiles of 256 x 256 or, where those are few, 128 x 128 with
// two workgroups a compute unit.  The last round's tiles are cut where that saves more
// than a part costs.  Measured: a step (64 elements) of a 256 x 256 tile 2.1 us, of two
// 128 x 128 tiles side by side 1.2; writing and adding their parts 26 and 13.  Of float32 (32
// elements) two 128 x 128 tiles 3.6, one of 64 rows 1.0, its parts 4.
struct HeadCut {
  bool big;
  int groups, whole, cuts;
  int64_t bytes;   // of the parts
};
template <class S>
static double head_cut_as(HeadCut& c, int64_t rows, int D, int K, int pairs, int cu) {
  constexpr bool kWide = sizeof(typename S::E) == 4;
  const double step = kWide ? S::TN == 64 ? 1.0 : 3.6 : S::TM == 256 ? 2.1 : 1.2;
  const double part = S::TM == 256 ? 26.0 : S::TN == 64 ? 4.0 : 13.0;
  const int64_t m = (D + S::TM - 1) / S::TM, n = (rows + S::TN - 1) / S::TN, tiles = m * n;
  const int64_t steps = (int64_t)pairs * ((K + S::kStep - 1) / S::kStep), at_once = (int64_t)cu * S::kPerCu;
  c.big = S::TM == 256;
  c.groups = (int)at_once;
  c.whole = (int)(tiles / at_once * at_once);
  c.cuts = 1;
  const int64_t rest = tiles - c.whole;
  double best = 0.0;
  if (rest > 0) {
    best = 1e30;
    for (int p = 1; p <= 64 && p * 4 <= steps + 3; ++p) {
      const double rounds = (double)((rest * p + at_once - 1) / at_once);
      const double time = rounds * (step * steps / p) + (p > 1 ? part * rest * p / at_once + 5.0 : 0.0);
      if (time < best) best = time, c.cuts = p;
    }
    if (c.whole == 0 && rest * c.cuts < at_once) c.groups = (int)(rest * c.cuts);
  }
  // (with uncut tiles the edge's lie behind `rest` unused ones)
  const int64_t parts = (c.cuts > 1 || D % S::TM != 0 ? rest * c.cuts : 0) + (D % S::TM == 0 ? 0 : n);
  c.bytes = parts * S::TM * S::TN * 4;
  return best + (double)(c.whole / at_once) * step * steps;
}
static bool head_few_back(int64_t N, bool native) { return native && N <= 64; }   // dz and dx
static HeadCut head_cut(int64_t rows, int D, int K, int pairs, bool native, bool few, int cu) {
  HeadCut big, mid;
  if (native) {
    if (few)
      head_cut_as<HeadFewBack>(mid, rows, D, K, pairs, cu);
    else
      head_cut_as<HeadMid<float>>(mid, rows, D, K, pairs, cu);
    return mid;
  }
  const double tb = head_cut_as<HeadBig<bf16>>(big, rows, D, K, pairs, cu);
  const double tm = head_cut_as<HeadMid<bf16>>(mid, rows, D, K, pairs, cu);
  return tb <= tm ? big : mid;
}
static int head_pair_count(int pa, int pb) { return pb == 1 ? 1 : pa == 1 ? 3 : 6; }
template <class S, bool BROWS>
static void head_grad_as(HeadGrad g, const HeadCut& c, hipStream_t s) {
  g.m_tiles = (g.D + S::TM - 1) / S::TM;
  g.n_tiles = (g.N + S::TN - 1) / S::TN;
  g.groups = c.groups;
  g.whole = c.whole;
  g.cuts = c.cuts;
  k_head_grad<S, BROWS><<<(unsigned)g.groups, S::kThreads, 0, s>>>(g);
  const int tiles = g.m_tiles * g.n_tiles, first = g.D % S::TM != 0 ? 0 : c.cuts > 1 ? c.whole : tiles;
  if (first < tiles) k_head_join_tiles<S, BROWS><<<dim3((unsigned)(tiles - first), 8), 256, 0, s>>>(g, first);
}
template <bool BROWS>
static void head_grad(const HeadGrad& g, bool native, int cu, hipStream_t s) {
  const bool few = BROWS && head_few_back(g.N, native);
  const HeadCut c = head_cut(g.N, g.D, g.pr.K, head_pair_count(g.pr.pa, g.pr.pb), native, few, cu);
  if constexpr (BROWS)
    if (few) return head_grad_as<HeadFewBack, true>(g, c, s);
  if (native)
    head_grad_as<HeadMid<float>, BROWS>(g, c, s);
  else if (c.big)
    head_grad_as<HeadBig<bf16>, BROWS>(g, c, s);
  else
    head_grad_as<HeadMid<bf16>, BROWS>(g, c, s);
}

// The backward's pieces of the vocabulary and its buffers
struct HeadPlan {
  int piece;            // tokens of a piece, a multiple of 256
  size_t dz, acc, part; // bytes
  size_t rest, sums, first, there, lists;   // of the targets' rests and tokens, and the rests' sums by token
  size_t bytes(const HeadLayout& l) const {
    return l.x_bytes + l.w_bytes + dz + acc + part + rest + sums + first + there + lists;
  }
};
static HeadPlan head_plan(int64_t N, int V, int D, const HeadLayout& l, bool x_bf16, int cu) {
  HeadPlan p;
  const int planes = l.px, pw = l.pw;
  const size_t size = l.native ? 4 : 2;
  const int64_t all = ((int64_t)V + 255) / 256 * 256;
  int64_t fit = (int64_t)(kHeadPiece / ((size_t)((N + 63) / 64 * 64) * size * planes)) / 256 * 256;
  fit = fit < 256 ? 256 : fit < kHeadPieceMost ? fit : kHeadPieceMost;
  const int64_t pieces = (all + fit - 1) / fit;
  p.piece = (int)(((all + pieces - 1) / pieces + 255) / 256 * 256);
  p.dz = up16((size_t)planes * ((N + 63) / 64 * 64) * p.piece * size);
  p.acc = all > p.piece && x_bf16 ? up16((size_t)N * D * 4) : 0;
  // the parts of dx and dW of a whole piece and of the last one
  const int last = (int)(V - (int64_t)(V - 1) / p.piece * p.piece);
  int64_t parts = 0;
  for (int vocab : {p.piece < V ? p.piece : V, last}) {
    const int64_t dx = head_cut(N, D, vocab, head_pair_count(pw, planes), l.native, head_few_back(N, l.native), cu).bytes;
    const int64_t dw = head_cut(vocab, D, (int)N, head_pair_count(planes, planes), l.native, false, cu).bytes;
    parts = dx > parts ? dx : parts;
    parts = dw > parts ? dw : parts;
  }
  p.part = (size_t)parts;
  p.rest = x_bf16 ? up16((size_t)N * 8) : 0;
  p.sums = x_bf16 ? up16((size_t)N * D * 2) : 0;
  p.first = x_bf16 ? up16((size_t)V * 4) : 0;
  p.there = x_bf16 ? up16((size_t)all / 8) : 0;
  p.lists = x_bf16 && N > kFewRows ? nsa_token_sums_workspace(N, D) : 0;
  return p;
}

}  // namespace nsa

// The workspaces cover any alignment of the operands: a packed copy where the
// dtypes or D alone need none is only made for pointers off 16 bytes.
extern "C" size_t nsa_head_fwd_workspace(int64_t N, int V, int D, int x_dtype, int w_dtype, int aligned, void* stream) {
  using namespace nsa;
  if (!head_shape_ok(N, V, D) || !head_type(x_dtype) || !head_type(w_dtype)) return 0;
  if (N == 0) return 16;
  const void* at = reinterpret_cast<const void*>(aligned ? 16 : 1);
  const int cu = device_cu_count(static_cast<hipStream_t>(stream));
  const HeadLayout l = head_layout(N, V, D, at, at, x_dtype, w_dtype, kNativeFwd, cu);
  const int split = head_as(head_fwd_kind(N, V, cu), l.native, [&](auto s) { return head_grid<decltype(s)>(N, V, cu).split; });
  return l.x_bytes + l.w_bytes + up16((size_t)split * N * sizeof(float2)) + (size_t)N * 4;
}

extern "C" int nsa_head_fwd(const void* x, const void* w, const int64_t* target, float* logp, float* lse,
                            void* workspace, size_t workspace_bytes, int64_t N, int V, int D, int x_dtype, int w_dtype,
                            void* stream) {
  using namespace nsa;
  NSA_CHECK(head_shape_ok(N, V, D), NSA_ERR_SHAPE);
  NSA_CHECK(head_type(x_dtype) && head_type(w_dtype), NSA_ERR_DTYPE);
  if (N == 0) return NSA_OK;
  NSA_CHECK(x != nullptr && w != nullptr && lse != nullptr && (target == nullptr) == (logp == nullptr), NSA_ERR_ARG);
  const hipStream_t s = static_cast<hipStream_t>(stream);
  const int cu = device_cu_count(s);
  const HeadLayout l = head_layout(N, V, D, x, w, x_dtype, w_dtype, kNativeFwd, cu);
  return head_as(head_fwd_kind(N, V, cu), l.native, [&](auto sh) -> int {
    using S = decltype(sh);
    const HeadGrid g = head_grid<S>(N, V, cu);
    NSA_CHECK(workspace != nullptr &&
                  workspace_bytes >= l.x_bytes + l.w_bytes + up16((size_t)g.split * N * sizeof(float2)) + (size_t)N * 4,
              NSA_ERR_WORKSPACE);
    NSA_CHECK(reinterpret_cast<uintptr_t>(workspace) % 16 == 0, NSA_ERR_ARG);
    char* ws = static_cast<char*>(workspace);
    char *const xp = ws, *const wp = ws + l.x_bytes;
    float2* part = reinterpret_cast<float2*>(ws + l.x_bytes + l.w_bytes);
    if (l.pack_x) head_pack(x, x_dtype, xp, N, D, l.ld, l.px, l.native, s);
    if (l.pack_w) head_pack(w, w_dtype, wp, V, D, l.ld, l.pw, l.native, s);
    HeadFwd a;
    a.pr.a = {l.pack_w ? wp : w, (int64_t)V * l.ld, l.pack_w ? l.ld : D, V, 0};
    a.pr.b = {l.pack_x ? xp : x, N * l.ld, l.pack_x ? l.ld : D, (int)N, 0};
    a.pr.K = D;
    a.pr.pa = l.pw;
    a.pr.pb = l.px;
    a.g = g;
    a.part = part;
    a.target = target;
    a.zt = reinterpret_cast<float*>(ws + l.x_bytes + l.w_bytes + up16((size_t)g.split * N * sizeof(float2)));
    a.N = (int)N;
    a.V = V;
    k_head_fwd<S><<<head_blocks(g), S::kThreads, 0, s>>>(a);
    const HeadJoin j{part, a.zt, target, logp, lse, N, g.split, V};
    k_head_join<<<(unsigned)((N + 3) / 4), 256, 0, s>>>(j);
    return nsa_launch_status();
  });
}

extern "C" size_t nsa_head_bwd_workspace(int64_t N, int V, int D, int x_dtype, int w_dtype, int aligned, void* stream) {
  using namespace nsa;
  if (!head_shape_ok(N, V, D) || !head_type(x_dtype) || !head_type(w_dtype)) return 0;
  if (N == 0) return 16;
  const void* at = reinterpret_cast<const void*>(aligned ? 16 : 1);
  const int cu = device_cu_count(static_cast<hipStream_t>(stream));
  const HeadLayout l = head_layout(N, V, D, at, at, x_dtype, w_dtype, kNativeBwd, cu);
  const HeadPlan p = head_plan(N, V, D, l, x_dtype == NSA_BF16, cu);
  return p.bytes(l);
}

extern "C" int nsa_head_bwd(const void* x, const void* w, const int64_t* target, const float* logp, const float* lse,
                            const float* dlogp, const float* dlse, void* dx, void* dw, void* workspace,
                            size_t workspace_bytes, int64_t N, int V, int D, int x_dtype, int w_dtype, void* stream) {
  using namespace nsa;
  NSA_CHECK(head_shape_ok(N, V, D) && N >= 1, NSA_ERR_SHAPE);
  NSA_CHECK(head_type(x_dtype) && head_type(w_dtype), NSA_ERR_DTYPE);
  NSA_CHECK(x != nullptr && w != nullptr && lse != nullptr && (dx != nullptr || dw != nullptr), NSA_ERR_ARG);
  NSA_CHECK(dlogp == nullptr || (target != nullptr && logp != nullptr), NSA_ERR_ARG);
  const hipStream_t s = static_cast<hipStream_t>(stream);
  const int cu = device_cu_count(s);
  const HeadLayout l = head_layout(N, V, D, x, w, x_dtype, w_dtype, kNativeBwd, cu);
  const HeadPlan p = head_plan(N, V, D, l, x_dtype == NSA_BF16, cu);
  NSA_CHECK(workspace != nullptr && workspace_bytes >= p.bytes(l), NSA_ERR_WORKSPACE);
  NSA_CHECK(reinterpret_cast<uintptr_t>(workspace) % 16 == 0, NSA_ERR_ARG);
  char* ws = static_cast<char*>(workspace);
  char* const xp = ws;
  ws += l.x_bytes;
  char* const wp = ws;
  ws += l.w_bytes;
  char* const dz = ws;
  ws += p.dz;
  float* acc = reinterpret_cast<float*>(ws);
  ws += p.acc;
  float* part = reinterpret_cast<float*>(ws);
  ws += p.part;
  float* rest = reinterpret_cast<float*>(ws);
  int* token = reinterpret_cast<int*>(rest + N);
  ws += p.rest;
  char* const sums = ws;
  ws += p.sums;
  int* first = reinterpret_cast<int*>(ws);
  ws += p.first;
  uint64_t* there = reinterpret_cast<uint64_t*>(ws);
  ws += p.there;
  if (l.pack_x) head_pack(x, x_dtype, xp, N, D, l.ld, l.px, l.native, s);
  if (l.pack_w) head_pack(w, w_dtype, wp, V, D, l.ld, l.pw, l.native, s);
  const unsigned rows = (unsigned)((N + 255) / 256);
  // the targets' rests come with the targets' elements of the first piece
  const bool rests = x_dtype == NSA_BF16 && dlogp != nullptr, few = rests && N <= kFewRows;
  const int ldx = l.pack_x ? l.ld : D, ldw = l.pack_w ? l.ld : D;
  const void* X = l.pack_x ? xp : x;
  const char* W = l.pack_w ? wp : static_cast<const char*>(w);
  const int64_t x_plane = N * (int64_t)l.ld, w_plane = (int64_t)V * l.ld, z_plane = (N + 63) / 64 * 64 * (int64_t)p.piece;
  for (int v0 = 0; v0 < V; v0 += p.piece) {
    const int vocab = V - v0 < p.piece ? V - v0 : p.piece;
    HeadDz z;
    z.pr.a = {W + (int64_t)v0 * ldw * (l.native ? 4 : 2), w_plane, ldw, vocab, 0};
    z.pr.b = {X, x_plane, ldx, (int)N, 0};
    z.pr.K = D;
    z.pr.pa = l.pw;
    z.pr.pb = l.px;
    z.lse = lse;
    z.dlogp = dlogp;
    z.dlse = dlse;
    z.target = target;
    z.dz = dz;
    z.ld = p.piece;
    z.plane = z_plane;
    z.N = (int)N;
    z.V = V;
    z.v0 = v0;
    z.vocab = vocab;
    z.rows = (int)((N + 63) / 64 * 64);
    auto form = [&](auto sh) {   // (its tiles cover dz's rows of zeros)
      using S = decltype(sh);
      z.g = head_grid<S>(N, vocab, cu);
      if constexpr (sizeof(typename S::E) == 2)
        if (l.px == 3) return k_head_dz<S, 3><<<head_blocks(z.g), S::kThreads, 0, s>>>(z);
      k_head_dz<S, 1><<<head_blocks(z.g), S::kThreads, 0, s>>>(z);
    };
    if (head_few_back(N, l.native))
      form(HeadFewBack{});
    else if (l.native)
      form(HeadMid<float>{});
    else if (head_kind(N, vocab, cu) == kBig)
      form(HeadBig<bf16>{});
    else
      form(HeadMid<bf16>{});
    if (few && v0 == 0) {
      bf16* const out = dw != nullptr ? reinterpret_cast<bf16*>(sums) : nullptr;
      const HeadFewRows f{z, logp, static_cast<const bf16*>(x), rest, token, out, first, there, D};
      const int64_t own = (N + kFewWaves - 1) / kFewWaves;
      const int64_t bits = dw != nullptr ? ((int64_t)V + kFewBits - 1) / kFewBits : 0;
      k_head_few<<<(unsigned)(own > bits ? own : bits), kFewThreads, 0, s>>>(f);
    } else if (l.native) {
      k_head_target<float, 1><<<rows, 256, 0, s>>>(z, logp, nullptr, nullptr);
    } else if (l.px == 3) {
      k_head_target<bf16, 3><<<rows, 256, 0, s>>>(z, logp, nullptr, nullptr);
    } else {
      const bool all = rests && v0 == 0;
      k_head_target<bf16, 1><<<rows, 256, 0, s>>>(z, logp, all ? rest : nullptr, token);
      if (all && dw != nullptr) {
        const int rc = nsa_token_sums(target, rest, x, sums, first, there, ws, N, V, D, stream);
        if (rc != NSA_OK) return rc;
      }
    }
    if (dx != nullptr) {
      HeadGrad g;
      const bool last = v0 + vocab >= V, lone = p.acc == 0;
      g.pr = {{W + (int64_t)v0 * ldw * (l.native ? 4 : 2), w_plane, ldw, ldw, vocab}, {dz, z_plane, p.piece, (int)N, 0}, vocab, l.pw, l.px};
      g.out = last || lone ? dx : static_cast<void*>(acc);
      g.out_bf16 = last && x_dtype == NSA_BF16;
      g.add = v0 == 0 ? nullptr : lone ? static_cast<const float*>(dx) : acc;
      g.part = part;
      g.N = (int)N;
      g.D = D;
      g.more = {rests && last ? reinterpret_cast<const bf16*>(W) : nullptr, ldw, token, rest, nullptr, nullptr};
      head_grad<true>(g, l.native, cu, s);
    }
    if (dw != nullptr) {
      HeadGrad g;
      g.pr = {{X, x_plane, ldx, ldx, (int)N}, {dz, z_plane, p.piece, p.piece, z.rows}, (int)N, l.px, l.px};
      g.out = static_cast<char*>(dw) + (int64_t)v0 * D * (w_dtype == NSA_BF16 ? 2 : 4);
      g.out_bf16 = w_dtype == NSA_BF16;
      g.add = nullptr;
      g.part = part;
      g.N = vocab;
      g.D = D;
      g.more = {rests ? reinterpret_cast<const bf16*>(sums) : nullptr, D, nullptr, nullptr, first + v0, there + v0 / 64};
      head_grad<false>(g, l.native, cu, s);
    }
  }
  return nsa_launch_status();
}
