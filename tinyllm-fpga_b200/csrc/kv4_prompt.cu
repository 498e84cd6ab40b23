// kv4_prompt.cu -- attention of prompts over the 4-bit paged KV cache: 256
// rows (query heads of one KV head times tokens) against blocks of 128
// positions on the tensor-memory MMAs.  Formulas, rounding and the joining of
// cut items as in kv4_attn.cu.
//
// Two tiles of 128 rows share every decoded key and value.  Of the CTA's
// warps, 4 + 4 are the tiles' softmax (one thread a row: no shuffles), 4 turn
// cached nibbles into operands in shared memory, and one thread a tile issues
// its MMAs: S = Q K^T into tensor memory, P = 2^k exp(s - max) written over S as
// the binary16 A operand of O += P V.  While one tile is in its softmax, the
// tensor core works for the other.
//
// What bounds it.  8192 tokens, 32 / 8 heads of 128, bfloat16, causal: 550 GFLOP
// in 657 us, 837 TFLOP/s (50% of the measured matrix product).  A block of 128
// positions costs 2048 cycles of MMAs (64 each, measured alone) and 2048 of the
// special function units (256 x 128 exponentials, 16 a cycle): both run at 41% to
// 45%.  The rest is the chain of a row's softmax between two waits, and an item's
// start and end.  With neither softmax nor decoding the first form took 715 us of
// its 863: waits beside busy MMAs take some 300 cycles.  At heads of 64 the MMAs
// are half and the softmax the same: 584 us.  binary16 (two operands of weights,
// twice the output MMAs) takes 1023 us.
// Tried: operands under the hardware's swizzle (decoding writes cost more
// addresses: 925 us against 863); one warp for both tiles' MMAs (818 against 713
// with one a tile); one lane polling the barriers for its warp (1075: slower).
//
// Waits are bounded.  When one runs out its CTA stops its work, waits for the
// MMAs in flight, marks the rows that it owes with NaN (a cut item's by the sum
// that its joining divides by) and leaves a note from which the joining launch
// makes the call's status.
//
// Order.  A tile's MMAs come from one thread, and the scores that overwrite a P
// are issued behind the product that reads it: the tensor pipe takes them in turn.
//
// Operand order.  A key word holds the dim pairs (n, n + 4), a value word the
// positions (i, i + 4): the contraction axes are taken in that order (0 4 1 5 2
// 6 3 7 of every 8), in Q and in P alike, so that decoding needs no
// rearrangement.  Operands lie as 8-row x 16-byte core matrices without
// swizzle: [contraction / 8][row][8], which the decoding lanes write 16 bytes
// at a time to 8 different bank groups.
#include "kv4_attn.cuh"

namespace bfp {
namespace kv4 {
namespace {

constexpr int PR = 256, PB = 128;            // rows of an item, positions of a block (of keys and values in shared memory)
constexpr int PU = 64;                       // positions of a unit: one MMA group of scores, one softmax step
constexpr int MIN_SHARE = 8;                 // blocks that are not worth a second CTA
// An item's queries, first block and outputs, in blocks (8192 tokens, 32 / 8
// heads of 128: 730 us at 3, 646 at 6, 666 at 9).
constexpr int ITEM = 6;
constexpr int THREADS = 512;                  // softmax 2 x 4 warps, decoding 4, MMA 2 (and 2 that wait at the end)

__device__ __forceinline__ void mb_init(unsigned long long* bar, unsigned count) {
  asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" :: "r"(su32(bar)), "r"(count) : "memory");
}
__device__ __forceinline__ void mb_arrive(unsigned long long* bar) {
  asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" :: "r"(su32(bar)) : "memory");
}
__device__ __forceinline__ bool mb_try(unsigned long long* bar, unsigned parity) {
  unsigned ok;
  asm volatile("{\n .reg .pred p;\n mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n selp.u32 %0, 1, 0, p;\n}\n"
               : "=r"(ok) : "r"(su32(bar)), "r"(parity) : "memory");
  return ok != 0;
}
// Shared-memory descriptor of a K-major operand without swizzle: low word
// start >> 4 [0,14), LBO >> 4 [16,30); high word SBO >> 4 (128 bytes) [0,14),
// version 1 at 14.  A step along the contraction adds to the low word.
constexpr uint32_t DESC_HI = (128u >> 4) | (1u << 14);
__device__ __forceinline__ uint32_t desc_lo(unsigned addr, unsigned lbo) { return (addr >> 4) | ((lbo >> 4) << 16); }
// kind::f16 instruction descriptor: D f32 [4,6)=1, A and B [7,10), [10,13) 0 f16 / 1 bf16,
// both K-major, N >> 3 at [17,23), M >> 4 at [24,29)
__host__ __device__ constexpr uint32_t idesc_f16(int bf, int M, int N) {
  return (1u << 4) | ((uint32_t)bf << 7) | ((uint32_t)bf << 10) | ((uint32_t)(N >> 3) << 17) | ((uint32_t)(M >> 4) << 24);
}
__device__ __forceinline__ void mma_ss(uint32_t d, uint32_t a, uint32_t b, uint32_t idesc, uint32_t add) {
  asm volatile("{\n .reg .pred p;\n .reg .b64 da, db;\n setp.ne.b32 p, %4, 0;\n mov.b64 da, {%1, %5};\n mov.b64 db, {%2, %5};\n"
               " tcgen05.mma.cta_group::1.kind::f16 [%0], da, db, %3, p;\n}\n"
               :: "r"(d), "r"(a), "r"(b), "r"(idesc), "r"(add), "r"(DESC_HI) : "memory");
}
__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t a, uint32_t b, uint32_t idesc, uint32_t add) {
  asm volatile("{\n .reg .pred p;\n .reg .b64 db;\n setp.ne.b32 p, %4, 0;\n mov.b64 db, {%2, %5};\n"
               " tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], db, %3, p;\n}\n"
               :: "r"(d), "r"(a), "r"(b), "r"(idesc), "r"(add), "r"(DESC_HI) : "memory");
}
__device__ __forceinline__ bool elect_one() {
  unsigned p;
  asm volatile("{\n .reg .pred p;\n elect.sync _|p, 0xffffffff;\n selp.u32 %0, 1, 0, p;\n}\n" : "=r"(p));
  return p != 0;
}
__device__ __forceinline__ void tc_commit(unsigned long long* bar) {
  asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" :: "r"(su32(bar)) : "memory");
}
__device__ __forceinline__ void tc_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tc_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void wait_ld() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void ld32(uint32_t at, uint32_t* r) {
  asm volatile("tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,"
               "%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
                 "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]),
                 "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]),
                 "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
               : "r"(at) : "memory");
}
__device__ __forceinline__ void st32(uint32_t at, const uint32_t* r) {
  asm volatile("tcgen05.st.sync.aligned.32x32b.x32.b32 [%32], {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,"
               "%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31};"
               :: "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]),
                  "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]),
                  "r"(r[16]), "r"(r[17]), "r"(r[18]), "r"(r[19]), "r"(r[20]), "r"(r[21]), "r"(r[22]), "r"(r[23]),
                  "r"(r[24]), "r"(r[25]), "r"(r[26]), "r"(r[27]), "r"(r[28]), "r"(r[29]), "r"(r[30]), "r"(r[31]),
                  "r"(at) : "memory");
}
// ---- the split: as in kv4_attn.cu, but under a causal mask or a window every
// row tile has its own number of blocks.  The functions are a warp's.
constexpr int CH = 256;
struct Plan {
  long long pre[CH + 1];                     // blocks before each sequence, or chunk of `per` sequences
  long long total, geff, delta;
  Span span[CH];                             // the sequences, where per == 1
  long long items;
  int per;
};
struct PSeq : Span { int rt, seq; };         // row tiles, index
struct Tiles { int first, nb; };             // first block of a row tile, its blocks plus ITEM

__device__ __forceinline__ PSeq seq_make(const AttnArgs& a, int s, const Span& p) {
  PSeq r;
  static_cast<Span&>(r) = p;
  r.seq = s;
  r.rt = (int)(((long long)p.n_q * a.group + PR - 1) / PR);
  return r;
}
__device__ __forceinline__ PSeq seq_at(const AttnArgs& a, int s) { return seq_make(a, s, span_of(a.b, s)); }
__device__ __forceinline__ Tiles tiles_of(const AttnArgs& a, const PSeq& q, int rt) {
  const int qp0 = q.qp0;
  const int j0 = (int)((long long)rt * PR / a.group), j1 = (int)min((long long)q.n_q - 1, ((long long)rt * PR + PR - 1) / a.group);
  const int hi = qp0 + j1 < 0 ? 0 : a.causal ? min(q.len, qp0 + j1 + 1) : q.len;
  const long long lo = a.window ? max(0LL, (long long)qp0 + j0 - a.window + 1) : 0;
  Tiles t;
  t.first = (int)min(lo / PB, (long long)(max(hi - 1, 0) / PB));
  t.nb = max((hi + PB - 1) / PB - t.first, 1) + ITEM;
  return t;
}
// Blocks of one head's row tiles [0, rt), summed by the warp.
__device__ __forceinline__ long long head_blocks(const AttnArgs& a, const PSeq& q) {
  long long n = 0;
  for (int r = threadIdx.x & 31; r < q.rt; r += 32) n += tiles_of(a, q, r).nb;
  #pragma unroll
  for (int o = 16; o; o >>= 1) n += __shfl_xor_sync(0xffffffffu, n, o);
  return n;
}

__device__ __forceinline__ void make_plan(const AttnArgs& a, Plan& s) {
  const int per = (a.b.n_seq + CH - 1) / CH, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (threadIdx.x == 0) { s.items = 0; s.per = per; }
  __syncthreads();
  // few sequences: a warp each; many (then short) ones: a thread each
  const bool wide = a.b.n_seq <= 32;
  for (int c = wide ? warp : (int)threadIdx.x; c < CH; c += wide ? THREADS / 32 : THREADS) {
    long long w = 0, items = 0;
    for (int i = c * per; i < min((c + 1) * per, a.b.n_seq); ++i) {
      const PSeq q = seq_at(a, i);
      if (per == 1) s.span[c] = q;
      long long n = 0;
      if (wide) n = head_blocks(a, q);
      else for (int r = 0; r < q.rt; ++r) n += tiles_of(a, q, r).nb;
      w += n * a.b.H;
      items += (long long)q.rt * a.b.H;
    }
    if (!wide || lane == 0) {
      s.pre[c + 1] = w;
      if (items) atomicAdd(reinterpret_cast<unsigned long long*>(&s.items), (unsigned long long)items);
    }
  }
  __syncthreads();
  if (warp == 0) {
    constexpr int C = CH / 32;
    long long v[C], sum = 0;
    #pragma unroll
    for (int i = 0; i < C; ++i) { sum += s.pre[lane * C + i + 1]; v[i] = sum; }
    long long inc = sum;
    #pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const long long y = __shfl_up_sync(0xffffffffu, inc, o);
      if (lane >= o) inc += y;
    }
    #pragma unroll
    for (int i = 0; i < C; ++i) s.pre[lane * C + i + 1] = inc - sum + v[i];
    if (lane == 31) {
      s.pre[0] = 0;
      s.total = inc;
      s.geff = max(min((long long)a.grid, max(s.items, (inc + MIN_SHARE - 1) / MIN_SHARE)), 1LL);
      s.delta = max(inc / (s.geff * 64), (long long)(ITEM + 1));   // no cut leaves less than a block
    }
  }
  __syncthreads();
}

struct PItem {
  PSeq q;
  int head, rt;                              // KV head, row tile
  Tiles t;
  long long start, end;
};

// A CTA's part of an item: blocks x .. xe - 1 of the schedule, n real ones from
// block blk0 of the sequence; blocks and segments before it (of both tiles, of
// the second), for the barriers' phases.
struct Seg {
  PItem it;
  long long x, xe;
  int r0, rows, n, blk0, nk, nt1, seg0, seg1;
};

// The item that holds block x (0 <= x < total); every lane of the warp calls with the same x.
__device__ __forceinline__ PItem item_of(const AttnArgs& a, const Plan& s, long long x) {
  const int lane = threadIdx.x & 31;
  int lo = 0, hi = CH;
  #pragma unroll 1
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (s.pre[mid] <= x) lo = mid; else hi = mid;
  }
  PItem it;
  long long at = s.pre[lo], w1;
  if (s.per == 1) {
    it.q = seq_make(a, lo, s.span[lo]);
    w1 = div_small(s.pre[lo + 1] - at, a.b.H);
  } else {
    for (int i = lo * s.per;; ++i) {
      it.q = seq_at(a, i);
      w1 = head_blocks(a, it.q);
      if (x < at + w1 * a.b.H || i + 1 >= a.b.n_seq) break;
      at += w1 * a.b.H;
    }
  }
  it.head = (int)div_small(x - at, max(w1, 1LL));
  at += it.head * w1;
  for (int r0 = 0;; r0 += 32) {                             // row tiles, 32 at a time
    const Tiles t = r0 + lane < it.q.rt ? tiles_of(a, it.q, r0 + lane) : Tiles{0, 0};
    int inc = t.nb;
    #pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int y = __shfl_up_sync(0xffffffffu, inc, o);
      if (lane >= o) inc += y;
    }
    const int sum = __shfl_sync(0xffffffffu, inc, 31);
    if (x < at + sum || r0 + 32 >= it.q.rt) {
      const unsigned here = __ballot_sync(0xffffffffu, x < at + inc);
      const int k = here ? __ffs(here) - 1 : 0;
      it.rt = r0 + k;
      it.t.first = __shfl_sync(0xffffffffu, t.first, k);
      it.t.nb = __shfl_sync(0xffffffffu, t.nb, k);
      it.end = at + __shfl_sync(0xffffffffu, inc, k);
      it.start = it.end - it.t.nb;
      return it;
    }
    at += sum;
  }
}

__device__ __forceinline__ long long bound_of(const AttnArgs& a, const Plan& s, long long i) {
  const long long x = div_small(i * s.total, s.geff);
  if (x <= 0 || x >= s.total) return x <= 0 ? 0 : s.total;
  const PItem it = item_of(a, s, x);
  const long long before = x - it.start, after = it.end - x;
  if (before <= after) return before <= s.delta ? it.start : x;
  return after <= s.delta ? it.end : x;
}

// The exponent scale of a binary16 pair whose nibbles all lie in bits 0..3.
struct ScaleV { unsigned s, c; };
__device__ __forceinline__ ScaleV scale_v(unsigned bytes) {
  const __half2 h = as_h2(bytes << 10);
  ScaleV r;
  r.s = as_u(__hmul2(h, __floats2half2_rn(0x1p-10f, 0x1p-10f)));
  r.c = as_u(__hmul2(h, __floats2half2_rn(-1032.f * 0x1p-10f, -1032.f * 0x1p-10f)));
  return r;
}

// Two 32-bit operations in one instruction.
__device__ __forceinline__ uint64_t pack2(float x, float y) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(x), "f"(y));
  return r;
}
__device__ __forceinline__ float2 unpack2(uint64_t v) {
  float2 r;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(v));
  return r;
}
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t d;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(a), "l"(b), "l"(c));
  return d;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
  uint64_t d;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
  return d;
}

// Scores of columns from `at` that the row does not see become -inf.
template <int N>
__device__ __forceinline__ void hide(uint32_t (&s)[N], int at, int lo, int hi) {
  #pragma unroll
  for (int k = 0; k < N; ++k) s[k] = at + k < hi && at + k >= lo ? s[k] : 0xFF800000u;
}

// P = ex2(scale s - ref) of a row's 64 scores, as MMA operand (of every 16
// columns the 8 words, then the 8 of its low part); returns their sum.
template <int PS>
__device__ __forceinline__ float row_weights(uint32_t (&ph)[32 * PS], const uint32_t (&s)[64], float scale, float ref) {
  const uint64_t sl = pack2(scale, scale), rf = pack2(-ref, -ref);
  uint64_t add[2] = {0, 0};
  #pragma unroll
  for (int c = 0; c < 4; ++c) {
    float p[16];
    #pragma unroll
    for (int k = 0; k < 16; k += 2) {
      const float2 y = unpack2(fma2(pack2(__uint_as_float(s[c * 16 + k]), __uint_as_float(s[c * 16 + k + 1])), sl, rf));
      p[k] = ex2(y.x);
      p[k + 1] = ex2(y.y);
      add[(k >> 1) & 1] = add2(add[(k >> 1) & 1], pack2(p[k], p[k + 1]));
    }
    #pragma unroll
    for (int k = 0; k < 8; ++k) {
      const int ia = (k >> 2) * 8 + (k & 3), ib = ia + 4;
      const __half2 h = __floats2half2_rn(p[ia], p[ib]);
      ph[c * 8 * PS + k] = as_u(h);
      if constexpr (PS == 2) {
        const float2 back = __half22float2(h);
        ph[c * 16 + 8 + k] = as_u(__floats2half2_rn(p[ia] - back.x, p[ib] - back.y));
      }
    }
  }
  const float2 t0 = unpack2(add[0]), t1 = unpack2(add[1]);
  return (t0.x + t0.y) + (t1.x + t1.y);
}

template <int HD> constexpr int SMEM = 2 * 128 * HD * 2 + 4 * PB * HD * 2;   // queries of two tiles, two stages of keys and of values

template <typename T, int HD>
__global__ void __launch_bounds__(THREADS, 1) prompt_kernel(const AttnArgs a, int spin, int q_vec, int o_vec) {
  constexpr int KU = HD / 32, REC9 = HD * 9 / 8, PS = Kind<T>::PS;
  constexpr bool HALF_K = Kind<T>::HALF_K;
  constexpr int TILE_Q = 128 * HD * 2, TILE_KV = PB * HD * 2;
  extern __shared__ __align__(128) unsigned char smem[];
  unsigned char *s_q = smem, *s_k = smem + 2 * TILE_Q, *s_v = s_k + 2 * TILE_KV;
  __shared__ Plan plan;
  __shared__ unsigned long long kfull[2], kfree[2], vfull[2], vfree[2], sfull[2][2], pfull[2][2], ofull[2][2], qfull[2], drained;
  __shared__ uint32_t s_tmem;
  __shared__ volatile int s_abort;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  if (tid == 0) {
    for (int i = 0; i < 2; ++i) {
      mb_init(&kfull[i], 4); mb_init(&kfree[i], 2); mb_init(&vfull[i], 4); mb_init(&vfree[i], 2);
      mb_init(&sfull[i][0], 1); mb_init(&sfull[i][1], 1); mb_init(&pfull[i][0], 4); mb_init(&pfull[i][1], 4); mb_init(&ofull[i][0], 1); mb_init(&ofull[i][1], 1); mb_init(&qfull[i], 4);
    }
    mb_init(&drained, 2);
    s_abort = 0;
    a.cuts[blockIdx.x] = Cut{};
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 12) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" :: "r"(su32(&s_tmem)), "r"(512) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  tc_before();
  make_plan(a, plan);                                       // (its barriers publish the above)
  tc_after();
  const uint32_t tmem = s_tmem;
  const auto wait = [&](unsigned long long* bar, unsigned parity) -> bool {
    for (int it = 0; it < spin; ++it) {
      if (mb_try(bar, parity)) return true;
      if (s_abort) return false;
    }
    s_abort = 1;
    return false;
  };

  // by a whole warp: one answer for all of its lanes
  const auto warp_wait = [&](unsigned long long* bar, unsigned parity) { return __all_sync(0xffffffffu, wait(bar, parity)) != 0; };

  const int page = a.b.page, rec_bytes = page * REC9;
  const long long page_bytes = (long long)rec_bytes * a.b.H;
  bool ok = true;
  // A CTA's share, item by item; every role walks through it by itself, also
  // when a wait has run out (!ok): then there are still rows to be marked.
  const auto share = [&](auto role) {
    if ((long long)blockIdx.x >= plan.geff || plan.total == 0) return;
    Seg g;
    g.nk = g.nt1 = g.seg0 = g.seg1 = 0;
    g.x = bound_of(a, plan, blockIdx.x);
    const long long x1 = bound_of(a, plan, (long long)blockIdx.x + 1);
    while (g.x < x1) {
      g.it = item_of(a, plan, g.x);
      g.xe = min(x1, g.it.end);
      if (g.xe <= g.x) break;                                // lengths changed during the call
      g.r0 = g.it.rt * PR;
      g.rows = (int)min((long long)PR, (long long)g.it.q.n_q * a.group - g.r0);
      const int skip = g.x == g.it.start ? 0 : (int)(g.x - g.it.start) - ITEM;   // blocks of CTAs before this one
      g.n = (int)(g.xe - g.it.start) - ITEM - skip;
      g.blk0 = g.it.t.first + skip;
      role(g);
      ok = __all_sync(0xffffffffu, ok);
      const bool two = g.rows > 128;
      g.nk += g.n;
      ++g.seg0;
      if (two) { g.nt1 += g.n; ++g.seg1; }
      g.x = g.xe;
    }
  };
  // what a row of the segment sees: positions lo .. hi - 1
  const auto hi_at = [&](const Seg& g, int j) {
    const int p = g.it.q.qp0 + j;
    return p < 0 ? 0 : a.causal ? min(g.it.q.len, p + 1) : g.it.q.len;
  };
  const auto lo_at = [&](const Seg& g, int j) {
    return a.window ? (int)max(0LL, (long long)g.it.q.qp0 + j - a.window + 1) : 0;
  };

  if (warp < 8) {
    // ================= softmax: one thread a row
    asm volatile("setmaxnreg.inc.sync.aligned.u32 160;");
    const auto part_of = [&](const Seg& g) { return a.part + ((long long)blockIdx.x * 2 + (g.x > g.it.start ? 0 : 1)) * PR * (HD + 2); };
    // a row that a wait left undone: NaN, in its output or in the sum that its joining divides by
    const auto not_done = [&](const Seg& g, int row, int token, int head) {
      if (g.x == g.it.start && g.xe == g.it.end) {
        T* dst = static_cast<T*>(a.out) + (long long)token * a.o_ts + (long long)head * a.o_hs;
        #pragma unroll 1
        for (int d = 0; d < HD; ++d) dst[d] = from_f<T>(NAN);
        if (a.lse) a.lse[(long long)token * a.HQ + head] = NAN;
      } else {
        float* part = part_of(g);
        part[PR * HD + row] = -INFINITY;
        part[PR * HD + PR + row] = NAN;
      }
    };
    share([&](const Seg& g) {
      const int tile = warp >> 2, n = g.n, blk0 = g.blk0, r0 = g.r0, rows = g.rows;
      if (tile == 0 || rows > 128) {
        const int row = tid & 127, R = r0 + tile * 128 + row, j = R / a.group;
        const bool live = tile * 128 + row < rows;
        const int q0 = g.it.q.q0, head = g.it.head * a.group + R - j * a.group;
        const uint32_t tq = (uint32_t)(32 * (warp & 3)) << 16;
        const uint32_t tS = tmem + tq + tile * 128, tO = tmem + tq + 256 + tile * HD;
        const int blocks0 = tile ? g.nt1 : g.nk, seg = tile ? g.seg1 : g.seg0;
        // queries: [dim / 8][row][dims 0 4 1 5 2 6 3 7]
        const T* q = static_cast<const T*>(a.q) + (long long)(q0 + j) * a.q_ts + (long long)head * a.q_hs;
        if (!ok) {
          if (live) not_done(g, tile * 128 + row, q0 + j, head);
          return;
        }
        uint4 qv[HD / 8];
        #pragma unroll
        for (int c = 0; c < HD / 8; ++c) {                  // (all of the row's loads at once)
          qv[c] = make_uint4(0, 0, 0, 0);
          if (live) {
            if (q_vec) {
              qv[c] = __ldg(reinterpret_cast<const uint4*>(q + c * 8));
            } else {
              unsigned short e[8];
              #pragma unroll
              for (int i = 0; i < 8; ++i) e[i] = __ldg(reinterpret_cast<const unsigned short*>(q) + c * 8 + i);
              qv[c] = make_uint4(e[0] | e[1] << 16, e[2] | e[3] << 16, e[4] | e[5] << 16, e[6] | e[7] << 16);
            }
          }
        }
        #pragma unroll
        for (int c = 0; c < HD / 8; ++c) {
          uint4 v = qv[c];
          v.x ^= a.q_flip; v.y ^= a.q_flip; v.z ^= a.q_flip; v.w ^= a.q_flip;
          *reinterpret_cast<uint4*>(s_q + tile * TILE_Q + c * 2048 + row * 16) =
              make_uint4(prmt(v.x, v.z, 0x5410), prmt(v.x, v.z, 0x7632), prmt(v.y, v.w, 0x5410), prmt(v.y, v.w, 0x7632));
        }
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        tc_before();                                        // (orders the last item's reads of O)
        __syncwarp();
        if (lane == 0) mb_arrive(&qfull[tile]);
        const int hi = live ? hi_at(g, j) : 0, lo = lo_at(g, j);
        const int ja = (r0 + tile * 128) / a.group, jb = (r0 + min(rows, tile * 128 + 128) - 1) / a.group;
        const int all_hi = hi_at(g, ja), all_lo = lo_at(g, jb);
        float m = -INFINITY, ref = 0.f, l = 0.f;
        for (int u = 0; u < 2 * n; ++u) {
          const int base = blk0 * PB + u * PU;
          const bool whole = base + PU <= all_hi && base >= all_lo;
          const uint32_t tU = tS + (u & 1) * PU;
          if (!(ok = warp_wait(&sfull[tile][u & 1], (blocks0 + (u >> 1)) & 1))) break;
          tc_after();
          uint32_t s[PU];
          ld32(tU, s);
          ld32(tU + 32, s + 32);
          wait_ld();
          if (!whole) hide(s, base, lo, hi);
          // The weights by the present reference, beside the maximum that tells
          // whether it still serves (one unit in many it does not).
          uint32_t ph[32 * PS];
          float sum = row_weights<PS>(ph, s, a.scale_log2, ref);
          float top[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
          #pragma unroll
          for (int k = 0; k < PU; k += 2) top[(k >> 1) & 3] = fmaxf(top[(k >> 1) & 3], fmaxf(__uint_as_float(s[k]), __uint_as_float(s[k + 1])));
          top[0] = fmaxf(fmaxf(top[0], top[1]), fmaxf(top[2], top[3]));
          if (__any_sync(0xffffffffu, top[0] > m + a.slack[PS - 1])) {
            const float mn = fmaxf(m, top[0]);
            const float al = mn == -INFINITY ? 1.f : ex2((m - mn) * a.scale_log2);
            m = mn;
            ref = mn == -INFINITY ? 0.f : mn * a.scale_log2 - P_EXP<PS>;
            l *= al;
            if (u > 0) {
              // the outputs of unit u - 1 are complete when the scores of unit u + 1 are, which follow them
              if (!(ok = u + 1 < 2 * n ? warp_wait(&sfull[tile][(u + 1) & 1], (blocks0 + ((u + 1) >> 1)) & 1) : warp_wait(&ofull[tile][0], seg & 1))) break;
              tc_after();
              #pragma unroll 1
              for (int c = 0; c < HD / 32; ++c) {
                uint32_t o[32];
                ld32(tO + c * 32, o);
                wait_ld();
                #pragma unroll
                for (int k = 0; k < 32; ++k) o[k] = __float_as_uint(__uint_as_float(o[k]) * al);
                st32(tO + c * 32, o);
              }
            }
            sum = row_weights<PS>(ph, s, a.scale_log2, ref);
          }
          l += sum;
          st32(tU, ph);
          if constexpr (PS == 2) st32(tU + 32, ph + 32);
          wait_st();
          tc_before();
          __syncwarp();
          if (lane == 0) mb_arrive(&pfull[tile][u & 1]);
        }
        if (ok && (ok = warp_wait(&ofull[tile][1], seg & 1))) {
          tc_after();
          const bool full = g.x == g.it.start && g.xe == g.it.end;
          const float inv = l == 0.f ? 0.f : V_UP / l;
          T* dst = static_cast<T*>(a.out) + (long long)(q0 + j) * a.o_ts + (long long)head * a.o_hs;
          float* part = part_of(g);
          const int pr = tile * 128 + row;
          #pragma unroll 1
          for (int c = 0; c < HD / 32; ++c) {
            uint32_t o[32];
            __syncwarp();
            ld32(tO + c * 32, o);
            wait_ld();
            if (live && full) {
              float f[32];
              #pragma unroll
              for (int k = 0; k < 32; ++k) f[k] = __uint_as_float(o[k]) * inv;
              if (o_vec) store_vec<T, 32, true>(dst + c * 32, f);
              else store_vec<T, 32, false>(dst + c * 32, f);
            } else if (live) {
              #pragma unroll
              for (int k = 0; k < 32; k += 4)
                *reinterpret_cast<uint4*>(part + (long long)pr * HD + c * 32 + k) = make_uint4(o[k], o[k + 1], o[k + 2], o[k + 3]);
            }
          }
          if (live && full && a.lse)
            a.lse[(long long)(q0 + j) * a.HQ + head] = l == 0.f ? -INFINITY : (m * a.scale_log2 + log2f(l) - P_EXP<PS>) * LN2;
          if (live && !full) {
            part[PR * HD + pr] = m * a.scale_log2;
            part[PR * HD + PR + pr] = l;
          }
        } else if (live) {
          not_done(g, tile * 128 + row, q0 + j, head);
        }
      }
    });
  } else if (warp < 12) {
    // ================= cached nibbles to operands: 32 positions of the block a warp
    asm volatile("setmaxnreg.inc.sync.aligned.u32 136;");
    share([&](const Seg& g) {
      const int n = g.n, blk0 = g.blk0, nk = g.nk;
      const int wd = warp - 8;
      const Magic mg = magic_numbers();
      constexpr int NKE = KU % 2 == 0 ? KU / 2 : KU, NVE = KU == 3 ? 3 : 1;
      const int kq = lane >> 2, kp = lane & 3, vo = lane >> 3, vp = lane & 7;   // quad and part of the keys; oct and part of the values
      const int any_lo = lo_at(g, g.r0 / a.group), v_hi = hi_at(g, (g.r0 + g.rows - 1) / a.group);
      const int seq_off = g.it.head * rec_bytes;
      const int* bt = a.b.bt + (long long)g.it.q.seq * a.b.bt_ld;
      uint4 k0[KU], v0[KU];
      unsigned ke[NKE];
      uint2 ve[NVE];
      const auto page_at = [&](int pos) -> int {
        const int i = pos >> a.b.page_shift;
        return i < a.b.max_pages ? __ldg(bt + i) : -1;
      };
      const uint4 zero = make_uint4(0x88888888u, 0x88888888u, 0x88888888u, 0x88888888u);
      const auto fetch_k = [&](int base, int pk) {
        const int at = (base + 32 * wd + 4 * kq) & (page - 1);
        const bool good = (unsigned)pk < (unsigned)a.b.n_pages;
        const uint8_t* rec = a.b.pool + (good ? pk * page_bytes : 0) + seq_off;
        #pragma unroll
        for (int w = 0; w < KU; ++w)
          k0[w] = good ? __ldg(reinterpret_cast<const uint4*>(rec + ((at >> 2) * (HD / 8) + kp * KU + w) * 16)) : zero;
        #pragma unroll
        for (int w = 0; w < NKE; ++w)
          ke[w] = good ? __ldg(reinterpret_cast<const unsigned*>(rec + page * HD + (NKE == KU ? (kp * KU + w) / 2 : kp * NKE + w) * page + at)) : 0x01010101u;
      };
      const auto fetch_v = [&](int base, int pv) {
        const int at = (base + 32 * wd + 8 * vo) & (page - 1);
        const bool good = (unsigned)pv < (unsigned)a.b.n_pages;
        const uint8_t* rec = a.b.pool + (good ? pv * page_bytes : 0) + seq_off;
        #pragma unroll
        for (int w = 0; w < KU; ++w) {
          const int u = KU == 2 || KU == 4 ? (w + vp) & (KU - 1) : w;
          v0[w] = good ? __ldg(reinterpret_cast<const uint4*>(rec + page * HD / 2 + ((at >> 3) * (HD / 4) + vp * KU + u) * 16)) : zero;
        }
        #pragma unroll
        for (int w = 0; w < NVE; ++w)
          ve[w] = good ? __ldg(reinterpret_cast<const uint2*>(rec + page * HD + (HD / 16 + (vp * KU + w) / 4) * page + at)) : make_uint2(0x01010101u, 0x01010101u);
      };
      // values at positions that no row sees: 0, whatever the bytes
      const auto clear_v = [&](int base) {
        #pragma unroll
        for (int w = 0; w < NVE; ++w)
          #pragma unroll
          for (int i = 0; i < 8; ++i) {
            const int p = base + 32 * wd + 8 * vo + i;
            if (p >= v_hi || p < any_lo) (i < 4 ? ve[w].x : ve[w].y) &= ~(0xFFu << (8 * (i & 3)));
          }
      };
      const int b0 = blk0 * PB + 32 * wd;
      fetch_k(blk0 * PB, page_at(b0 + 4 * kq));
      fetch_v(blk0 * PB, page_at(b0 + 8 * vo));
      int pk = -1, pv = -1;
      if (n > 1) { pk = page_at(b0 + PB + 4 * kq); pv = page_at(b0 + PB + 8 * vo); }
      for (int i = 0; i < n && ok; ++i) {
        const int kc = nk + i, st = kc & 1;
        // keys
        if (kc >= 2 && !(ok = warp_wait(&kfree[st], ((kc >> 1) + 1) & 1))) break;
        #pragma unroll
        for (int w = 0; w < KU; ++w) {
          unsigned r[4] = {k0[w].x, k0[w].y, k0[w].z, k0[w].w};
          // position (i + part) & 3 at step i: 8 lanes then write to 8 bank groups
          if (kp & 1) { const unsigned f = r[0]; r[0] = r[1]; r[1] = r[2]; r[2] = r[3]; r[3] = f; }
          if (kp & 2) { unsigned f = r[0]; r[0] = r[2]; r[2] = f; f = r[1]; r[1] = r[3]; r[3] = f; }
          const unsigned eb = __funnelshift_r(ke[NKE == KU ? w : w / 2], ke[NKE == KU ? w : w / 2], 8 * kp);
          unsigned char* d = s_k + st * TILE_KV + (kp * KU + w) * 2048 + (32 * wd + 4 * kq) * 16;
          #pragma unroll
          for (int p = 0; p < 4; ++p) {
            unsigned o[4];
            const KeyScaleT<HALF_K> sc = key_scale<HALF_K>(prmt(eb, 0u, p | 0x40 | p << 8 | 0x4000));
            key_pairs<HALF_K>(mg, r[p], sc, o);
            *reinterpret_cast<uint4*>(d + ((p + kp) & 3) * 16) = make_uint4(o[0], o[1], o[2], o[3]);
          }
        }
        if (i + 1 < n) fetch_k((blk0 + i + 1) * PB, pk);    // (comes while the values are worked on)
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        __syncwarp();
        if (lane == 0) mb_arrive(&kfull[st]);
        // values
        if ((blk0 + i + 1) * PB > v_hi || (blk0 + i) * PB < any_lo) clear_v((blk0 + i) * PB);
        if (kc >= 2 && !(ok = warp_wait(&vfree[st], ((kc >> 1) + 1) & 1))) break;
        ScaleV sc[4];
        #pragma unroll
        for (int w = 0; w < KU; ++w) {
          const int u = KU == 2 || KU == 4 ? (w + vp) & (KU - 1) : w;
          if (w == 0 || NVE > 1) {
            #pragma unroll
            for (int p = 0; p < 4; ++p)
              sc[p] = scale_v(prmt(ve[NVE > 1 ? w : 0].x, ve[NVE > 1 ? w : 0].y, p * 0x0101 | 0x0080 | (4 + p) << 8 | (12 + p) << 12));
          }
          const unsigned word[4] = {v0[w].x, v0[w].y, v0[w].z, v0[w].w};
          unsigned char* d = s_v + st * TILE_KV + (4 * wd + vo) * (HD * 16) + (vp * KU + u) * 64;
          #pragma unroll
          for (int k = 0; k < 4; ++k) {
            const int nn = (k + (vp >> 1)) & 3;             // dim 4 u + nn
            unsigned o[4];
            #pragma unroll
            for (int p = 0; p < 4; ++p)
              o[p] = as_u(__hfma2(as_h2(and_or<0x000F000Fu>(word[p] >> (4 * nn), mg.h1024)), as_h2(sc[p].s), as_h2(sc[p].c)));
            *reinterpret_cast<uint4*>(d + nn * 16) = make_uint4(o[0], o[1], o[2], o[3]);
          }
        }
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        __syncwarp();
        if (lane == 0) mb_arrive(&vfull[st]);
        if (i + 1 < n) fetch_v((blk0 + i + 1) * PB, pv);
        if (i + 2 < n) { pk = page_at(b0 + (i + 2) * PB + 4 * kq); pv = page_at(b0 + (i + 2) * PB + 8 * vo); }
      }
      if (g.x == g.it.start && g.xe < g.it.end && warp == 9) {
        // the parts end at the last boundary below the item's end, unless that was moved onto it
        const long long c = blockIdx.x;
        long long e = min(plan.geff, div_small(g.it.end * plan.geff + plan.total - 1, plan.total));
        while (e - 1 > c + 1 && bound_of(a, plan, e - 1) >= g.it.end) --e;
        if (lane == 0) a.cuts[c] = Cut{(int)(e - c), g.it.q.q0, g.rows, g.r0, g.it.head * a.group, 0, {0, 0}};
      }
    });
  } else {
    // ================= the MMAs: a warp a tile waits together, one lane issues.
    // (A wait takes some 300 cycles beside MMAs that keep shared memory busy: one
    // tile's lie under the other's MMAs.)
    asm volatile("setmaxnreg.dec.sync.aligned.u32 56;");
    if (warp < 14) share([&](const Seg& g) {
      if (!ok) return;
      const int n = g.n, nk = g.nk, t = warp - 12;
      const bool both = g.rows > 128;
      if (t && !both) {
        // No tile of its own: it still gives back every block, so that it is never
        // ahead of the phases that it will wait for in a later item.
        for (int kc = nk; kc < nk + n; ++kc) {
          if (!(ok = warp_wait(&kfull[kc & 1], (kc >> 1) & 1))) return;
          if (lane == 0) mb_arrive(&kfree[kc & 1]);
          if (!(ok = warp_wait(&vfull[kc & 1], (kc >> 1) & 1))) return;
          if (lane == 0) mb_arrive(&vfree[kc & 1]);
        }
        return;
      }
      constexpr uint32_t i_qk = idesc_f16(HALF_K ? 0 : 1, 128, PU), i_pv = idesc_f16(0, 128, HD);
      const uint32_t tm = __shfl_sync(0xffffffffu, tmem, 0);
      const uint32_t tS = tm + t * 128, tO = tm + 256 + t * HD;
      const uint32_t dq = desc_lo(su32(s_q), 2048) + t * (TILE_Q >> 4), dk = desc_lo(su32(s_k), 2048), dv = desc_lo(su32(s_v), HD * 16);
      const int blocks0 = t ? g.nt1 : nk;
      // Scores run a unit ahead of the softmax: those of unit u + 2 follow the
      // outputs of unit u, whose weights lay in the same columns.
      const auto scores = [&](int u, int st) {              // by the issuing lane
        #pragma unroll
        for (int k = 0; k < HD / 16; ++k)
          mma_ss(tS + (u & 1) * PU, dq + k * 256, dk + st * (TILE_KV >> 4) + (u & 1) * (PU * 16 >> 4) + k * 256, i_qk, k > 0);
        tc_commit(&sfull[t][u & 1]);
      };
      ok = warp_wait(&qfull[t], (t ? g.seg1 : g.seg0) & 1) && warp_wait(&kfull[nk & 1], (nk >> 1) & 1);
      tc_after();
      if (ok && elect_one()) {
        scores(0, nk & 1);
        scores(1, nk & 1);
        tc_commit(&kfree[nk & 1]);                          // (two arrivals, one of each MMA warp)
      }
      __syncwarp();
      for (int u = 0; u < 2 * n && ok; ++u) {
        const int kc = nk + (u >> 1), st = kc & 1;
        const bool more = u + 2 < 2 * n;
        // the next block's keys come after this one's values
        if (!(u & 1) && !(ok = more ? warp_wait(&kfull[st ^ 1], ((kc + 1) >> 1) & 1) : warp_wait(&vfull[st], (kc >> 1) & 1))) break;
        if (!(ok = warp_wait(&pfull[t][u & 1], (blocks0 + (u >> 1)) & 1))) break;
        tc_after();
        if (elect_one()) {
          #pragma unroll
          for (int k = 0; k < PU / 16; ++k) {
            const uint32_t ap = tS + (u & 1) * PU + k * 8 * PS, bv = dv + st * (TILE_KV >> 4) + ((u & 1) * (PU / 16) + k) * 2 * HD;
            mma_ts(tO, ap, bv, i_pv, k > 0 || u > 0);
            if constexpr (PS == 2) mma_ts(tO, ap + 8, bv, i_pv, 1);
          }
          if (more) scores(u, st ^ 1);
          else tc_commit(&ofull[t][u & 1]);                 // the last two units'
          if (u & 1) {
            tc_commit(&vfree[st]);
            if (more) tc_commit(&kfree[st ^ 1]);
          }
        }
        __syncwarp();
      }
    });
  }
  __syncwarp();
  if (warp == 12 || warp == 13) {                           // every MMA has ended before the tensor memory goes back
    if (elect_one()) tc_commit(&drained);
    __syncwarp();
    for (int i = 0; i < SPIN && !mb_try(&drained, 0); ++i) {}
  }
  tc_before();
  __syncthreads();
  if (tid == 0) a.cuts[blockIdx.x].late = s_abort;
  if (warp == 12) {
    tc_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" :: "r"(tmem), "r"(512) : "memory");
  }
}

}  // namespace

size_t prompt_ws_bytes(int hd, int n_sm) { return sizeof(Status) + (size_t)n_sm * (sizeof(Cut) + 2 * PR * (hd + 2) * 4); }

template <typename T, int HD>
cudaError_t launch_prompt(AttnArgs a, int n_sm, int spin, void* ws, cudaStream_t s) {
  auto* kern = prompt_kernel<T, HD>;
  static std::atomic<unsigned char> allowed[128];
  cudaError_t e = allow_smem(kern, SMEM<HD>, allowed);
  if (e != cudaSuccess) return e;
  a.grid = n_sm;
  a.status = static_cast<Status*>(ws);
  a.cuts = reinterpret_cast<Cut*>(a.status + 1);
  a.part = reinterpret_cast<float*>(a.cuts + a.grid);
  const auto vec = [](const void* p, long long ts, long long hs) {
    return reinterpret_cast<uintptr_t>(p) % 16 == 0 && ts % 8 == 0 && hs % 8 == 0 ? 1 : 0;
  };
  kern<<<a.grid, THREADS, SMEM<HD>, s>>>(a, spin, vec(a.q, a.q_ts, a.q_hs), vec(a.out, a.o_ts, a.o_hs));
  e = cudaGetLastError();
  return e == cudaSuccess ? launch_join<T, HD, PR, true>(a, 16, s) : e;
}

#define BFP200_PROMPT(T) \
  template cudaError_t launch_prompt<T, 32>(AttnArgs, int, int, void*, cudaStream_t); \
  template cudaError_t launch_prompt<T, 64>(AttnArgs, int, int, void*, cudaStream_t); \
  template cudaError_t launch_prompt<T, 96>(AttnArgs, int, int, void*, cudaStream_t); \
  template cudaError_t launch_prompt<T, 128>(AttnArgs, int, int, void*, cudaStream_t);
BFP200_PROMPT(__nv_bfloat16)
BFP200_PROMPT(__half)

}  // namespace kv4
}  // namespace bfp
