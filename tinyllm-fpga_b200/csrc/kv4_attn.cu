// kv4_attn.cu -- attention over the 4-bit paged KV cache (record layout and
// number format in kv4.cuh).
//
//   o_r = sum_k w_rk v_k / sum_k w_rk,  w_rk = exp(scale q_r . k_k),  k over the positions that row r sees
//   lse_r = log sum_k w_rk
//
// One pass over the cache with the running maximum and sum of the softmax.
// The rows of one KV head (its query heads times the call's tokens) share
// every cached byte.  Both products run on mma.sync with the cache as the A
// operand and the rows as N: S^T[position][row] = K Q^T and O^T[dim][row] =
// V^T P^T, so that a group of up to 8 rows needs no padding to 16, and the
// cache goes from global memory to the A registers without shared memory:
// the record layout is the register layout (4 positions x 8 dims and 8
// positions x 4 dims of 16 bytes).  S^T's accumulators become P^T's operand by
// one 8x8 transpose (movmatrix) per 8 positions.
//
// Rounding.  K is exact in the operand type; Q is split into as many operands
// of that type as hold all its bits (1 for 16-bit types, 3 bfloat16 for
// 32-bit); V and P use binary16, in which V 2^-4 is exact and P = 2^15 exp(s
// - max) keeps 11 bits (bfloat16 results: an error of 2^-12 beside the
// result's own 2^-9), or 22 bits in two operands where the result is binary16
// or 32-bit.  Scores, maxima, sums and accumulators are 32-bit.
//
// Work split.  All (sequence, KV head, row tile) items are laid end to end in
// blocks of 32 positions and cut evenly over the CTAs on the device, from the
// lengths there; cuts near an item's end move onto it.  Cut items leave
// partial sums that a second, dependent launch joins in a fixed order.
#include "kv4.cuh"

#include <exception>
#include <string>
#include <type_traits>

int bfp200_set_error(int code, const std::string& msg);   // engine.cu

namespace bfp {
namespace kv4 {
namespace {

constexpr int BLK = 32;            // positions of one step of a warp
constexpr int MINB = 8;            // blocks that are not worth a second CTA
constexpr float LN2 = 0.6931471805599453f;
constexpr float P_EXP = 15.f;      // P is held times 2^15: subnormal only below 2^-29 of the maximum
constexpr float V_UP = 16.f;       // V is held times 2^-4

struct AttnArgs {
  Batch b;
  const void* q;
  void* out;
  float* lse;                      // [T][HQ] or null
  float* part;                     // partial sums: [CTA][2][NR][HD + 2]
  long long q_ts, q_hs, o_ts, o_hs;
  int HQ, group, causal;
  long long window;                // 0: none
  float scale_log2;
  int grid;                        // CTAs of the first launch
};

// ---- the split ---------------------------------------------------------------
struct Seq {
  int q0, n_q, len, blk0, nb, rt;  // first token, tokens, positions, first block, blocks, row tiles
};

template <int NR>
__device__ __forceinline__ Seq seq_of(const AttnArgs& a, int s) {
  Seq r;
  const int qs = min(max(__ldg(a.b.q_start + s), 0), a.b.T);
  const int qe = min(max(__ldg(a.b.q_start + s + 1), qs), a.b.T);
  r.q0 = qs;
  r.n_q = qe - qs;
  r.len = min(max(__ldg(a.b.lens + s), 0), a.b.max_pages << a.b.page_shift);
  const long long first = a.window ? (long long)r.len - r.n_q - a.window + 1 : 0;
  r.blk0 = first > 0 ? min((int)(first / BLK), max(r.len - 1, 0) / BLK) : 0;
  r.nb = max((r.len + BLK - 1) / BLK - r.blk0, 1);
  r.rt = (int)(((long long)r.n_q * a.group + NR - 1) / NR);
  return r;
}

constexpr int SCH = 128;           // chunks of sequences whose block counts are summed
struct Sched {
  long long pre[SCH + 1];          // blocks before each chunk
  long long total, geff, delta;
  int per;                         // sequences per chunk
};

// Fills the schedule; every thread of the CTA takes part.
template <int NR>
__device__ void make_sched(const AttnArgs& a, Sched& s, int n_thr) {
  __shared__ long long s_items;
  const int per = (a.b.n_seq + SCH - 1) / SCH;
  if (threadIdx.x == 0) s_items = 0;
  __syncthreads();
  long long items = 0;
  for (int c = threadIdx.x; c < SCH; c += n_thr) {
    long long w = 0;
    for (int i = c * per; i < min((c + 1) * per, a.b.n_seq); ++i) {
      const Seq q = seq_of<NR>(a, i);
      const long long n = (long long)q.rt * a.b.H;
      items += n;
      w += n * q.nb;
    }
    s.pre[c + 1] = w;
  }
  for (int o = 16; o; o >>= 1) items += __shfl_xor_sync(0xffffffffu, items, o);
  if ((threadIdx.x & 31) == 0 && items) atomicAdd(reinterpret_cast<unsigned long long*>(&s_items), (unsigned long long)items);
  __syncthreads();
  if (threadIdx.x < 32) {                                   // inclusive sums: 4 chunks a lane
    constexpr int C = SCH / 32;
    long long v[C], sum = 0;
    #pragma unroll
    for (int i = 0; i < C; ++i) { sum += s.pre[threadIdx.x * C + i + 1]; v[i] = sum; }
    long long inc = sum;
    #pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const long long y = __shfl_up_sync(0xffffffffu, inc, o);
      if ((int)threadIdx.x >= o) inc += y;
    }
    #pragma unroll
    for (int i = 0; i < C; ++i) s.pre[threadIdx.x * C + i + 1] = inc - sum + v[i];
    if (threadIdx.x == 31) {
      s.total = inc;
      const long long want = max((long long)s_items, (inc + MINB - 1) / MINB);
      s.geff = max(min((long long)a.grid, want), 1LL);
      s.delta = max(inc / s.geff / 4, (long long)(MINB / 2));
      s.pre[0] = 0;
      s.per = per;
    }
  }
  __syncthreads();
}

struct Item {
  int seq, idx;                    // idx = head * rt + row tile
  long long start, end;            // its blocks
  Seq q;
};

// The item that holds block x (0 <= x < total).
template <int NR>
__device__ Item item_at(const AttnArgs& a, const Sched& s, long long x) {
  int lo = 0, hi = SCH;                                     // pre[lo] <= x < pre[hi]
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (s.pre[mid] <= x) lo = mid; else hi = mid;
  }
  Item it;
  long long at = s.pre[lo];
  it.seq = lo * s.per;
  for (;; ++it.seq) {
    it.q = seq_of<NR>(a, it.seq);
    const long long w = (long long)it.q.rt * a.b.H * it.q.nb;
    if (x < at + w || it.seq + 1 >= a.b.n_seq) break;
    at += w;
  }
  it.idx = (int)((x - at) / it.q.nb);
  it.start = at + (long long)it.idx * it.q.nb;
  it.end = it.start + it.q.nb;
  return it;
}

// First block of CTA i: an even share, moved onto an item's edge if one is near.
template <int NR>
__device__ long long bound(const AttnArgs& a, const Sched& s, long long i) {
  const long long x = i * s.total / s.geff;
  if (x <= 0 || x >= s.total) return x <= 0 ? 0 : s.total;
  const Item it = item_at<NR>(a, s, x);
  const long long before = x - it.start, after = it.end - x;
  if (before <= after) return before <= s.delta ? it.start : x;
  return after <= s.delta ? it.end : x;
}

// ---- arithmetic ------------------------------------------------------------------
__device__ __forceinline__ void mma_bf16(float (&c)[4], const unsigned (&a)[4], uint2 b) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
               : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
               : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b.x), "r"(b.y));
}
__device__ __forceinline__ void mma_f16(float (&c)[4], const unsigned (&a)[4], uint2 b) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
               : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
               : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b.x), "r"(b.y));
}
__device__ __forceinline__ unsigned transpose8(unsigned x) {
  unsigned y;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}
__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ unsigned as_u(__half2 h) { return *reinterpret_cast<unsigned*>(&h); }
__device__ __forceinline__ __half2 as_h2(unsigned u) { return *reinterpret_cast<__half2*>(&u); }
__device__ __forceinline__ unsigned as_u(__nv_bfloat162 h) { return *reinterpret_cast<unsigned*>(&h); }
__device__ __forceinline__ __nv_bfloat162 as_b2(unsigned u) { return *reinterpret_cast<__nv_bfloat162*>(&u); }

// Bytes of (a, b) by selector; 8 + n takes the sign of byte n, which is 0 for
// an exponent byte (__byte_perm has no such form).
__device__ __forceinline__ unsigned prmt(unsigned a, unsigned b, unsigned sel) {
  unsigned y;
  asm("prmt.b32 %0, %1, %2, %3;" : "=r"(y) : "r"(a), "r"(b), "r"(sel));
  return y;
}
// (x & mask) | magic in one instruction
template <unsigned MASK, unsigned MAGIC>
__device__ __forceinline__ unsigned and_or(unsigned x) {
  unsigned y;
  asm("lop3.b32 %0, %1, %2, %3, 0xEA;" : "=r"(y) : "r"(x), "n"(MASK), "n"(MAGIC));
  return y;
}

// Binary16 pairs of a word: nibbles (n, n + 4) under the scales (lo, hi) of
// its halves.  A nibble in bits 0..3 of 1024's fraction is 1024 + nibble, in
// bits 4..7 of 64's it is 64 + nibble; one multiply-add, exact, takes off
// 1024 + 8 or 64 + 8 and scales.
struct ScaleH { unsigned s, c1024, c64; };
__device__ __forceinline__ ScaleH scale_h(unsigned bytes) {       // exponent bytes in the low bytes of both halves
  const __half2 h = as_h2(bytes << 10);                             // 2^(B - 15)
  ScaleH r;                                                         // 2^(B - 25) = 2^-4 2^(B - 21)
  r.s = as_u(__hmul2(h, __floats2half2_rn(0x1p-10f, 0x1p-10f)));
  r.c1024 = as_u(__hmul2(h, __floats2half2_rn(-1032.f * 0x1p-10f, -1032.f * 0x1p-10f)));
  r.c64 = as_u(__hmul2(h, __floats2half2_rn(-72.f * 0x1p-10f, -72.f * 0x1p-10f)));
  return r;
}
template <int N>
__device__ __forceinline__ unsigned pair_h(unsigned w, unsigned w8, const ScaleH& sc) {   // w8 = w >> 8
  const unsigned src = N < 2 ? w : w8;
  const unsigned x = (N & 1) ? and_or<0x00F000F0u, 0x54005400u>(src) : and_or<0x000F000Fu, 0x64006400u>(src);
  return as_u(__hfma2(as_h2(x), as_h2(sc.s), as_h2((N & 1) ? sc.c64 : sc.c1024)));
}
// Bfloat16 pairs: 128 + nibble, less 136, scaled; exact.
struct ScaleB { unsigned s, c; };
__device__ __forceinline__ ScaleB scale_b(unsigned bytes) {
  ScaleB r;
  r.s = bytes * 128u + 0x35003500u;                                 // 2^(B - 21)
  r.c = as_u(__hmul2(as_b2(r.s), __floats2bfloat162_rn(-136.f, -136.f)));
  return r;
}
template <int N>
__device__ __forceinline__ unsigned pair_b(unsigned w, const ScaleB& sc) {
  const unsigned x = and_or<0x000F000Fu, 0x43004300u>(w >> (4 * N));
  return as_u(__hfma2(as_b2(x), as_b2(sc.s), as_b2(sc.c)));
}

template <typename T> struct Kind;
template <> struct Kind<__nv_bfloat16> { static constexpr int QS = 1, PS = 1; static constexpr bool HALF_K = false; };
template <> struct Kind<__half> { static constexpr int QS = 1, PS = 2; static constexpr bool HALF_K = true; };
template <> struct Kind<float> { static constexpr int QS = 3, PS = 2; static constexpr bool HALF_K = false; };

// The QS operands that add up to a pair of query values.
template <typename T>
__device__ __forceinline__ void split_q(T a, T b, unsigned (&o)[Kind<T>::QS]) {
  if constexpr (std::is_same<T, float>::value) {
    float x = a, y = b;
    #pragma unroll
    for (int i = 0; i < 3; ++i) {                                   // cut off 8 bits at a time; the rest is exact
      const unsigned hx = __float_as_uint(x) & 0xFFFF0000u, hy = __float_as_uint(y) & 0xFFFF0000u;
      o[i] = (hx >> 16) | hy;
      x = isfinite(x) ? x - __uint_as_float(hx) : 0.f;
      y = isfinite(y) ? y - __uint_as_float(hy) : 0.f;
    }
  } else {
    unsigned short ua, ub;
    memcpy(&ua, &a, 2);
    memcpy(&ub, &b, 2);
    o[0] = (unsigned)ua | ((unsigned)ub << 16);
  }
}

template <int HD>
struct Tile {                        // this lane's part of 32 positions
  static constexpr int KU = HD / 32;
  static constexpr int NKE = KU % 2 == 0 ? KU / 2 : KU;   // distinct exponent tiles of the lane's key units
  static constexpr int NVE = KU == 3 ? 3 : 1;             // ... of its value units
  uint4 k[KU], v[KU];
  unsigned ke[NKE];
  uint2 ve[NVE];
};

__device__ __forceinline__ uint4 ld16(const uint8_t* p) {
  uint4 r;
  asm volatile("ld.global.nc.L1::no_allocate.v4.u32 {%0,%1,%2,%3}, [%4];"
               : "=r"(r.x), "=r"(r.y), "=r"(r.z), "=r"(r.w) : "l"(p));
  return r;
}

template <typename T, int HD, int NT, int W>
__global__ void __launch_bounds__(W * 32) attn_kernel(const AttnArgs a) {
  constexpr int NR = NT * 8, KU = HD / 32, QS = Kind<T>::QS, PS = Kind<T>::PS, REC9 = HD * 9 / 8;
  constexpr bool HALF_K = Kind<T>::HALF_K;
  using TL = Tile<HD>;
  extern __shared__ __align__(16) unsigned char smem[];
  uint2* s_q = reinterpret_cast<uint2*>(smem);                        // [HD/16][NT][QS][32]
  float* s_o = reinterpret_cast<float*>(s_q + HD / 16 * NT * QS * 32);  // [W][NR][HD]
  float* s_m = s_o + W * NR * HD;                                     // [W][NR], [W][NR]
  float* s_l = s_m + W * NR;
  __shared__ Sched sch;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, t = lane & 3;
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  make_sched<NR>(a, sch, W * 32);
  if ((long long)blockIdx.x >= sch.geff || sch.total == 0) return;
  long long x = bound<NR>(a, sch, blockIdx.x);
  const long long x1 = bound<NR>(a, sch, (long long)blockIdx.x + 1);
  const int page = a.b.page, rec_bytes = page * REC9;
  Item it;
  if (x < x1) it = item_at<NR>(a, sch, x);
  while (x < x1) {
    const long long xe = min(x1, it.end);
    if (xe <= x) break;                                               // lengths changed during the call
    const int rt = it.q.rt, h = it.idx / rt, r0 = (it.idx - h * rt) * NR;
    const int rows = min(NR, it.q.n_q * a.group - r0);
    const int len = it.q.len, qp0 = len - it.q.n_q;                   // position of the sequence's first query
    // ---- rows: queries to operand registers
    for (int i = tid; i < HD / 16 * NT * 32; i += W * 32) {
      const int l = i & 31, nt = (i >> 5) % NT, st = i / (32 * NT);
      const int r = nt * 8 + (l >> 2), d = ((l & 3) * KU + (st >> 1)) * 8 + (st & 1) * 2;
      unsigned o0[QS], o1[QS];
      if (r < rows) {
        const int R = r0 + r, j = R / a.group;
        const T* p = static_cast<const T*>(a.q) + (long long)(it.q.q0 + j) * a.q_ts +
                     (long long)(h * a.group + R - j * a.group) * a.q_hs + d;
        split_q<T>(p[0], p[4], o0);
        split_q<T>(p[1], p[5], o1);
      } else {
        #pragma unroll
        for (int k = 0; k < QS; ++k) o0[k] = o1[k] = 0;
      }
      #pragma unroll
      for (int k = 0; k < QS; ++k) s_q[((st * NT + nt) * QS + k) * 32 + l] = make_uint2(o0[k], o1[k]);
    }
    // ---- what the rows see
    const int j0 = r0 / a.group, j1 = (r0 + rows - 1) / a.group;
    const auto hi_of = [&](int j) { return qp0 + j < 0 ? 0 : a.causal ? min(len, qp0 + j + 1) : len; };
    const auto lo_of = [&](int j) { return a.window ? (int)max(0LL, (long long)qp0 + j - a.window + 1) : 0; };
    const int all_hi = hi_of(j0), any_hi = hi_of(j1), all_lo = lo_of(j1), any_lo = lo_of(j0);
    int hi[NT][2], lo[NT][2];
    #pragma unroll
    for (int nt = 0; nt < NT; ++nt)
      #pragma unroll
      for (int c = 0; c < 2; ++c) {
        const int r = nt * 8 + 2 * t + c, j = (r0 + r) / a.group;
        hi[nt][c] = r < rows ? hi_of(j) : 0;
        lo[nt][c] = lo_of(j);
      }
    float m[NT][2], lsum[NT][2], O[KU][2][NT][4];
    #pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      m[nt][0] = m[nt][1] = -INFINITY;
      lsum[nt][0] = lsum[nt][1] = 0.f;
      #pragma unroll
      for (int w = 0; w < KU; ++w)
        #pragma unroll
        for (int n = 0; n < 2; ++n)
          #pragma unroll
          for (int k = 0; k < 4; ++k) O[w][n][nt][k] = 0.f;
    }
    __syncthreads();

    // this segment's blocks that some row sees, as positions
    const int first = max((int)(x - it.start) + it.q.blk0, any_lo / BLK);
    const int last = min((int)(xe - it.start) + it.q.blk0, (any_hi + BLK - 1) / BLK);
    const int* bt = a.b.bt + (long long)it.seq * a.b.bt_ld;
    const auto page_at = [&](int pos) -> int {
      const int i = pos >> a.b.page_shift;
      return i < a.b.max_pages ? __ldg(bt + i) : -1;
    };
    const auto load = [&](TL& tl, int base, int pk, int pv) {
      const int slot_k = (base + 4 * g) & (page - 1), slot_v = (base + 8 * t) & (page - 1);
      if ((unsigned)pk < (unsigned)a.b.n_pages) {
        const uint8_t* rec = a.b.pool + ((long long)pk * a.b.H + h) * rec_bytes;
        const uint8_t* kp = rec + ((slot_k >> 2) * (HD / 8) + t * KU) * 16;
        #pragma unroll
        for (int w = 0; w < KU; ++w) tl.k[w] = ld16(kp + w * 16);
        #pragma unroll
        for (int w = 0; w < TL::NKE; ++w) {
          const int tile = TL::NKE == KU ? (t * KU + w) / 2 : t * TL::NKE + w;
          tl.ke[w] = __ldg(reinterpret_cast<const unsigned*>(rec + page * HD + tile * page + slot_k));
        }
      } else {
        #pragma unroll
        for (int w = 0; w < KU; ++w) tl.k[w] = make_uint4(0x88888888u, 0x88888888u, 0x88888888u, 0x88888888u);
        #pragma unroll
        for (int w = 0; w < TL::NKE; ++w) tl.ke[w] = 0x01010101u;
      }
      if ((unsigned)pv < (unsigned)a.b.n_pages) {
        const uint8_t* rec = a.b.pool + ((long long)pv * a.b.H + h) * rec_bytes;
        const uint8_t* vp = rec + page * HD / 2 + ((slot_v >> 3) * (HD / 4) + g * KU) * 16;
        #pragma unroll
        for (int w = 0; w < KU; ++w) tl.v[w] = ld16(vp + w * 16);
        #pragma unroll
        for (int w = 0; w < TL::NVE; ++w) {
          const int tile = (g * KU + w) / 4;
          tl.ve[w] = __ldg(reinterpret_cast<const uint2*>(rec + page * HD + (HD / 16 + tile) * page + slot_v));
        }
      } else {
        #pragma unroll
        for (int w = 0; w < KU; ++w) tl.v[w] = make_uint4(0x88888888u, 0x88888888u, 0x88888888u, 0x88888888u);
        #pragma unroll
        for (int w = 0; w < TL::NVE; ++w) tl.ve[w] = make_uint2(0x01010101u, 0x01010101u);
      }
    };

    const auto compute = [&](const TL& tl, int base) {
      // ---- S^T = K Q^T: tiles of rows (position 4 g, 4 g + 1) and (4 g + 2, 4 g + 3)
      // (the query's low parts are summed apart: the tensor core cuts addends off at the sum's last bit)
      float S[2][NT][4], S_low[QS > 1 ? 2 : 1][QS > 1 ? NT : 1][4];
      #pragma unroll
      for (int i = 0; i < 2; ++i)
        #pragma unroll
        for (int nt = 0; nt < NT; ++nt)
          #pragma unroll
          for (int k = 0; k < 4; ++k) {
            S[i][nt][k] = 0.f;
            if constexpr (QS > 1) S_low[i][nt][k] = 0.f;
          }
      const auto keys = [&](auto W_) {
        constexpr int w = decltype(W_)::value;
        const unsigned word[4] = {tl.k[w].x, tl.k[w].y, tl.k[w].z, tl.k[w].w};
        const unsigned eb = tl.ke[TL::NKE == KU ? w : w / 2];
        unsigned op[4][4];                                       // [position][pair]
        #pragma unroll
        for (int i = 0; i < 4; ++i) {
          const unsigned by = __byte_perm(eb, 0, 0x4040 | (i * 0x0101));
          if constexpr (HALF_K) {
            const ScaleH sc = scale_h(by);
            const unsigned w8 = word[i] >> 8;
            op[i][0] = pair_h<0>(word[i], w8, sc);
            op[i][1] = pair_h<1>(word[i], w8, sc);
            op[i][2] = pair_h<2>(word[i], w8, sc);
            op[i][3] = pair_h<3>(word[i], w8, sc);
          } else {
            const ScaleB sc = scale_b(by);
            op[i][0] = pair_b<0>(word[i], sc);
            op[i][1] = pair_b<1>(word[i], sc);
            op[i][2] = pair_b<2>(word[i], sc);
            op[i][3] = pair_b<3>(word[i], sc);
          }
        }
        #pragma unroll
        for (int hf = 0; hf < 2; ++hf)
          #pragma unroll
          for (int nt = 0; nt < NT; ++nt)
            #pragma unroll
            for (int k = 0; k < QS; ++k) {
              const uint2 qb = s_q[(((w * 2 + hf) * NT + nt) * QS + k) * 32 + lane];
              #pragma unroll
              for (int i = 0; i < 2; ++i) {
                const unsigned fr[4] = {op[2 * i][2 * hf], op[2 * i + 1][2 * hf], op[2 * i][2 * hf + 1], op[2 * i + 1][2 * hf + 1]};
                if constexpr (HALF_K) mma_f16(S[i][nt], fr, qb);
                else if (k == 0) mma_bf16(S[i][nt], fr, qb);
                else mma_bf16(S_low[QS > 1 ? i : 0][QS > 1 ? nt : 0], fr, qb);
              }
            }
      };
      keys(std::integral_constant<int, 0>{});
      if constexpr (KU > 1) keys(std::integral_constant<int, 1>{});
      if constexpr (KU > 2) keys(std::integral_constant<int, 2>{});
      if constexpr (KU > 3) keys(std::integral_constant<int, 3>{});

      // ---- running softmax
      const bool whole = base + BLK <= all_hi && base >= all_lo;
      unsigned P[PS][4][NT];
      bool moved = false;
      float al[NT][2];
      #pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        float top[2];
        #pragma unroll
        for (int c = 0; c < 2; ++c) {
          #pragma unroll
          for (int i = 0; i < 4; ++i) {
            float& s = S[i >> 1][nt][(i & 1) * 2 + c];
            if constexpr (QS > 1) s += S_low[i >> 1][nt][(i & 1) * 2 + c];
            s *= a.scale_log2;
            if (!whole) {
              const int p = base + 4 * g + i;
              s = p < hi[nt][c] && p >= lo[nt][c] ? s : -INFINITY;
            }
          }
          top[c] = fmaxf(fmaxf(S[0][nt][c], S[0][nt][2 + c]), fmaxf(S[1][nt][c], S[1][nt][2 + c]));
          #pragma unroll
          for (int o = 4; o < 32; o <<= 1) top[c] = fmaxf(top[c], __shfl_xor_sync(0xffffffffu, top[c], o));
          const float mn = fmaxf(m[nt][c], top[c]);
          const float ref = mn == -INFINITY ? 0.f : mn;
          al[nt][c] = ex2(m[nt][c] - ref);
          moved |= mn != m[nt][c];
          m[nt][c] = mn;
          top[c] = ref - P_EXP;
        }
        float add[2] = {0.f, 0.f};
        #pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float p0 = ex2(S[i >> 1][nt][(i & 1) * 2] - top[0]), p1 = ex2(S[i >> 1][nt][(i & 1) * 2 + 1] - top[1]);
          add[0] += p0;
          add[1] += p1;
          const __half2 hp = __floats2half2_rn(p0, p1);
          P[0][i][nt] = transpose8(as_u(hp));
          if constexpr (PS == 2) {
            const float2 back = __half22float2(hp);
            P[1][i][nt] = transpose8(as_u(__floats2half2_rn(p0 - back.x, p1 - back.y)));
          }
        }
        lsum[nt][0] = lsum[nt][0] * al[nt][0] + add[0];
        lsum[nt][1] = lsum[nt][1] * al[nt][1] + add[1];
      }
      if (__any_sync(0xffffffffu, moved)) {
        #pragma unroll
        for (int w = 0; w < KU; ++w)
          #pragma unroll
          for (int n = 0; n < 2; ++n)
            #pragma unroll
            for (int nt = 0; nt < NT; ++nt)
              #pragma unroll
              for (int k = 0; k < 4; ++k) O[w][n][nt][k] *= al[nt][k & 1];
      }
      // ---- O^T += V^T P^T.  Bytes at positions that no row sees may be anything:
      // their scale becomes 0, which makes the values 0 and never NaN.
      const int v_hi = min(len, any_hi);
      const auto values = [&](auto W_) {
        constexpr int w = decltype(W_)::value;
        const unsigned word[4] = {tl.v[w].x, tl.v[w].y, tl.v[w].z, tl.v[w].w};
        const uint2 eb = tl.ve[TL::NVE == 1 ? 0 : w];
        #pragma unroll
        for (int j = 0; j < 2; ++j) {
          unsigned op[2][4];                                     // [pair of positions][dim]
          #pragma unroll
          for (int i2 = 0; i2 < 2; ++i2) {
            const int i = 2 * j + i2;
            unsigned by = prmt(eb.x, eb.y, (i | (8 + i) << 4 | (4 + i) << 8 | (12 + i) << 12));
            if (!whole) {
              const int p = base + 8 * t + i;
              if (p >= v_hi || p < any_lo) by &= 0xFFFF0000u;
              if (p + 4 >= v_hi || p + 4 < any_lo) by &= 0x0000FFFFu;
            }
            const ScaleH sc = scale_h(by);
            const unsigned w8 = word[i] >> 8;
            op[i2][0] = pair_h<0>(word[i], w8, sc);
            op[i2][1] = pair_h<1>(word[i], w8, sc);
            op[i2][2] = pair_h<2>(word[i], w8, sc);
            op[i2][3] = pair_h<3>(word[i], w8, sc);
          }
          #pragma unroll
          for (int n = 0; n < 2; ++n) {
            const unsigned fr[4] = {op[0][2 * n], op[0][2 * n + 1], op[1][2 * n], op[1][2 * n + 1]};
            #pragma unroll
            for (int nt = 0; nt < NT; ++nt)
              #pragma unroll
              for (int k = 0; k < PS; ++k) mma_f16(O[w][n][nt], fr, make_uint2(P[k][2 * j][nt], P[k][2 * j + 1][nt]));
          }
        }
      };
      values(std::integral_constant<int, 0>{});
      if constexpr (KU > 1) values(std::integral_constant<int, 1>{});
      if constexpr (KU > 2) values(std::integral_constant<int, 2>{});
      if constexpr (KU > 3) values(std::integral_constant<int, 3>{});
    };

    if (first + warp < last) {
      int blk = first + warp;
      TL cur, nxt;
      load(cur, blk * BLK, page_at(blk * BLK + 4 * g), page_at(blk * BLK + 8 * t));
      int pk = -1, pv = -1;
      if (blk + W < last) { pk = page_at((blk + W) * BLK + 4 * g); pv = page_at((blk + W) * BLK + 8 * t); }
      while (blk < last) {
        const int next = blk + W;
        if (next < last) {
          load(nxt, next * BLK, pk, pv);
          if (next + W < last) { pk = page_at((next + W) * BLK + 4 * g); pv = page_at((next + W) * BLK + 8 * t); }
        }
        compute(cur, blk * BLK);
        cur = nxt;
        blk = next;
      }
    }

    // ---- join the warps
    #pragma unroll
    for (int nt = 0; nt < NT; ++nt)
      #pragma unroll
      for (int c = 0; c < 2; ++c) {
        #pragma unroll
        for (int o = 4; o < 32; o <<= 1) lsum[nt][c] += __shfl_xor_sync(0xffffffffu, lsum[nt][c], o);
        const int r = nt * 8 + 2 * t + c;
        if (g == 0) { s_m[warp * NR + r] = m[nt][c]; s_l[warp * NR + r] = lsum[nt][c]; }
        #pragma unroll
        for (int w = 0; w < KU; ++w)
          #pragma unroll
          for (int n = 0; n < 2; ++n)
            *reinterpret_cast<float2*>(s_o + (warp * NR + r) * HD + (g * KU + w) * 4 + 2 * n) =
                make_float2(O[w][n][nt][c], O[w][n][nt][2 + c]);
      }
    __syncthreads();
    const bool full = x == it.start && xe == it.end;
    float* part = a.part + ((long long)blockIdx.x * 2 + (x > it.start ? 0 : 1)) * NR * (HD + 2);
    for (int i = tid; i < rows * (HD / 4); i += W * 32) {
      const int r = i / (HD / 4), d = (i - r * (HD / 4)) * 4;
      float M = s_m[r];
      #pragma unroll
      for (int w = 1; w < W; ++w) M = fmaxf(M, s_m[w * NR + r]);
      const float ref = M == -INFINITY ? 0.f : M;
      float L = 0.f;
      float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
      #pragma unroll
      for (int w = 0; w < W; ++w) {
        const float f = ex2(s_m[w * NR + r] - ref);
        const float4 v = *reinterpret_cast<const float4*>(s_o + (w * NR + r) * HD + d);
        L += s_l[w * NR + r] * f;
        o.x += v.x * f; o.y += v.y * f; o.z += v.z * f; o.w += v.w * f;
      }
      if (full) {
        const int R = r0 + r, j = R / a.group, head = h * a.group + R - j * a.group;
        const float inv = L == 0.f ? 0.f : V_UP / L;
        T* dst = static_cast<T*>(a.out) + (long long)(it.q.q0 + j) * a.o_ts + (long long)head * a.o_hs + d;
        dst[0] = from_f<T>(o.x * inv);
        dst[1] = from_f<T>(o.y * inv);
        dst[2] = from_f<T>(o.z * inv);
        dst[3] = from_f<T>(o.w * inv);
        if (d == 0 && a.lse) a.lse[(long long)(it.q.q0 + j) * a.HQ + head] = L == 0.f ? -INFINITY : (M + log2f(L) - P_EXP) * LN2;
      } else {
        *reinterpret_cast<float4*>(part + r * HD + d) = o;
        if (d == 0) { part[NR * HD + r] = M; part[NR * HD + NR + r] = L; }
      }
    }
    __syncthreads();
    // ---- the next item
    x = xe;
    if (x < x1) {
      if (it.idx + 1 < it.q.rt * a.b.H) {
        ++it.idx;
        it.start = it.end;
        it.end += it.q.nb;
      } else {
        it = item_at<NR>(a, sch, x);
      }
    }
  }
}

// Joins the partial sums of the items that CTA boundary blockIdx.x cuts first.
template <typename T, int HD, int NT>
__global__ void __launch_bounds__(128) join_kernel(const AttnArgs a) {
  constexpr int NR = NT * 8, Q = HD / 4, NG = 128 / Q;          // NG groups of threads share the parts
  __shared__ Sched sch;
  __shared__ float4 s_o[NG][Q];
  __shared__ float s_m[NG], s_l[NG];
  make_sched<NR>(a, sch, 128);
  const long long i = (long long)blockIdx.x + 1;
  long long x = 0;
  Item it;
  bool mine = i < sch.geff && sch.total > 0;
  if (mine) {
    x = bound<NR>(a, sch, i);
    mine = x < sch.total;
    if (mine) {
      it = item_at<NR>(a, sch, x);
      mine = x > it.start && bound<NR>(a, sch, i - 1) <= it.start;
    }
  }
  if (!mine) return;
  long long i_end = i + 1;                                       // CTAs i - 1 .. i_end - 1 hold parts
  while (i_end < sch.geff && bound<NR>(a, sch, i_end) < it.end) ++i_end;
  const int n = (int)(i_end - i) + 1;
  const int rt = it.q.rt, h = it.idx / rt, r0 = (it.idx - h * rt) * NR, rows = min(NR, it.q.n_q * a.group - r0);
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const int grp = threadIdx.x / Q, d4 = threadIdx.x % Q;
  for (int r = blockIdx.y; r < rows; r += gridDim.y) {
    float M = -INFINITY, L = 0.f;
    float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
    if (grp < NG) {
      #pragma unroll 4
      for (int k = grp; k < n; k += NG) {
        const long long cta = i - 1 + k;
        const float* part = a.part + (cta * 2 + (k ? 0 : 1)) * NR * (HD + 2);
        const float mk = __ldcg(part + NR * HD + r), lk = __ldcg(part + NR * HD + NR + r);
        const float4 v = __ldcg(reinterpret_cast<const float4*>(part + r * HD) + d4);
        const float mn = fmaxf(M, mk), ref = mn == -INFINITY ? 0.f : mn;
        const float fo = ex2(M - ref), fk = ex2(mk - ref);
        L = L * fo + lk * fk;
        o.x = o.x * fo + v.x * fk; o.y = o.y * fo + v.y * fk;
        o.z = o.z * fo + v.z * fk; o.w = o.w * fo + v.w * fk;
        M = mn;
      }
      s_o[grp][d4] = o;
      if (d4 == 0) { s_m[grp] = M; s_l[grp] = L; }
    }
    __syncthreads();
    if (grp == 0) {
      float mm = s_m[0];
      #pragma unroll
      for (int k = 1; k < NG; ++k) mm = fmaxf(mm, s_m[k]);
      const float ref = mm == -INFINITY ? 0.f : mm;
      L = 0.f;
      o = make_float4(0.f, 0.f, 0.f, 0.f);
      #pragma unroll
      for (int k = 0; k < NG; ++k) {
        const float f = ex2(s_m[k] - ref);
        const float4 v = s_o[k][d4];
        L += s_l[k] * f;
        o.x += v.x * f; o.y += v.y * f; o.z += v.z * f; o.w += v.w * f;
      }
      const int R = r0 + r, j = R / a.group, head = h * a.group + R - j * a.group;
      const float inv = L == 0.f ? 0.f : V_UP / L;
      T* dst = static_cast<T*>(a.out) + (long long)(it.q.q0 + j) * a.o_ts + (long long)head * a.o_hs + d4 * 4;
      dst[0] = from_f<T>(o.x * inv);
      dst[1] = from_f<T>(o.y * inv);
      dst[2] = from_f<T>(o.z * inv);
      dst[3] = from_f<T>(o.w * inv);
      if (d4 == 0 && a.lse) a.lse[(long long)(it.q.q0 + j) * a.HQ + head] = L == 0.f ? -INFINITY : (mm + log2f(L) - P_EXP) * LN2;
    }
    __syncthreads();
  }
}

template <int NT> constexpr int warps_of() { return NT == 4 ? 4 : 8; }

template <typename T, int HD, int NT>
cudaError_t launch_attn(AttnArgs a, int n_sm, float* ws, cudaStream_t s) {
  constexpr int W = warps_of<NT>(), NR = NT * 8;
  constexpr size_t smem = (size_t)(HD / 16) * NT * Kind<T>::QS * 32 * 8 + (size_t)W * NR * (HD + 2) * 4;
  static_assert(smem <= 200 * 1024, "shared memory");
  auto* kern = attn_kernel<T, HD, NT, W>;
  cudaError_t e;
  if (smem > 48 * 1024) {
    e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
    if (e != cudaSuccess) return e;
  }
  a.grid = n_sm * (512 / (W * 32));
  a.part = ws;
  kern<<<a.grid, W * 32, smem, s>>>(a);
  e = cudaGetLastError();
  if (e != cudaSuccess) return e;
  // items of at most MINB blocks are never cut
  if ((long long)a.b.max_pages * a.b.page <= MINB * BLK) return cudaSuccess;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(a.grid - 1, NR < 8 ? NR : 8);
  cfg.blockDim = dim3(128);
  cfg.stream = s;
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = at;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, join_kernel<T, HD, NT>, a);
}

// Row tile of a call: the sequences' average of tokens times the group.
int pick_nt(const Batch& b, int group) {
  const long long rows = ((long long)b.T + b.n_seq - 1) / b.n_seq * group;
  return rows <= 8 ? 1 : rows <= 16 ? 2 : 4;
}
// Room for the partial sums of any call with this head dim.
size_t ws_bytes(int hd, int n_sm) {
  size_t most = 0;
  for (int nt = 1; nt <= 4; nt *= 2) {
    const size_t grid = (size_t)n_sm * (512 / ((nt == 4 ? 4 : 8) * 32)), b = grid * 2 * nt * 8 * (hd + 2) * 4;
    most = b > most ? b : most;
  }
  return most;
}

template <typename T, int HD>
cudaError_t by_nt(const AttnArgs& a, int nt, int n_sm, float* ws, cudaStream_t s) {
  return nt == 1 ? launch_attn<T, HD, 1>(a, n_sm, ws, s)
       : nt == 2 ? launch_attn<T, HD, 2>(a, n_sm, ws, s)
                 : launch_attn<T, HD, 4>(a, n_sm, ws, s);
}
template <typename T>
cudaError_t by_hd(int hd, const AttnArgs& a, int nt, int n_sm, float* ws, cudaStream_t s) {
  return hd == 32 ? by_nt<T, 32>(a, nt, n_sm, ws, s)
       : hd == 64 ? by_nt<T, 64>(a, nt, n_sm, ws, s)
       : hd == 96 ? by_nt<T, 96>(a, nt, n_sm, ws, s)
                  : by_nt<T, 128>(a, nt, n_sm, ws, s);
}

}  // namespace
}  // namespace kv4
}  // namespace bfp

using namespace bfp::kv4;

extern "C" int bfp200_kv4_attention_workspace(const bfp200_kv4_attention_args* in, size_t* bytes) {
  const char* who = "kv4_attention_workspace";
  const auto bad = [&](const char* what) { return bfp200_set_error(BFP200_EINVAL, std::string(who) + ": " + what); };
  if (!in || !bytes) return bad("no arguments");
  Batch b;
  if (int rc = fill_batch(in->batch, &b, who)) return rc;
  if (in->H_Q < 1 || in->H_Q % b.H) return bad("H_Q must be a positive multiple of H_KV");
  int n_sm = 0;
  if (int rc = device_ready(who, &n_sm)) return rc;
  *bytes = ws_bytes((int)in->batch.HD, n_sm);
  return BFP200_OK;
}

extern "C" int bfp200_kv4_attention_dev(const bfp200_kv4_attention_args* in, void* stream) try {
  const char* who = "kv4_attention_dev";
  const auto bad = [&](const char* what) { return bfp200_set_error(BFP200_EINVAL, std::string(who) + ": " + what); };
  if (!in) return bad("no arguments");
  const bfp200_kv4_attention_args& r = *in;
  AttnArgs a;
  if (int rc = fill_batch(r.batch, &a.b, who)) return rc;
  const int es = r.dtype == BFP200_F32 ? 4 : r.dtype == BFP200_F16 || r.dtype == BFP200_BF16 ? 2 : 0;
  if (!es) return bad("dtype must be BFP200_F32, BFP200_F16 or BFP200_BF16");
  if (r.H_Q < 1 || r.H_Q > (1LL << 16) || r.H_Q % a.b.H) return bad("H_Q must be a positive multiple of H_KV");
  if (r.window < 0) return bad("window must not be negative");
  if (!(r.scale - r.scale == 0.0)) return bad("scale must be finite");
  if (a.b.T == 0 || a.b.n_seq == 0) return BFP200_OK;
  if (!r.q_dev || !r.out_dev) return bad("null pointer");
  if ((reinterpret_cast<uintptr_t>(r.q_dev) | reinterpret_cast<uintptr_t>(r.out_dev)) % es ||
      reinterpret_cast<uintptr_t>(r.lse_dev) % 4 || reinterpret_cast<uintptr_t>(r.workspace_dev) % 16)
    return bad("misaligned pointer");
  int n_sm = 0;
  if (int rc = device_ready(who, &n_sm)) return rc;
  a.q = r.q_dev; a.out = r.out_dev; a.lse = r.lse_dev;
  a.q_ts = r.q_ts; a.q_hs = r.q_hs; a.o_ts = r.o_ts; a.o_hs = r.o_hs;
  a.HQ = (int)r.H_Q;
  a.group = a.HQ / a.b.H;
  a.causal = r.causal != 0;
  a.window = r.window;
  a.scale_log2 = (float)(r.scale * 1.4426950408889634 * (r.dtype == BFP200_F16 ? 16.0 : 1.0));   // K is held times 2^-4 there
  a.grid = 0;
  a.part = nullptr;
  const int nt = pick_nt(a.b, a.group), hd = (int)r.batch.HD;
  if (!r.workspace_dev || r.workspace_bytes < (long long)ws_bytes(hd, n_sm))
    return bad("the workspace is smaller than bfp200_kv4_attention_workspace says");
  float* ws = static_cast<float*>(r.workspace_dev);
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const cudaError_t e = r.dtype == BFP200_F32 ? by_hd<float>(hd, a, nt, n_sm, ws, s)
                      : r.dtype == BFP200_F16 ? by_hd<__half>(hd, a, nt, n_sm, ws, s)
                                              : by_hd<__nv_bfloat16>(hd, a, nt, n_sm, ws, s);
  if (e != cudaSuccess) return bfp200_set_error(BFP200_ECUDA, std::string(who) + ": " + cudaGetErrorString(e));
  return BFP200_OK;
} catch (const std::exception& ex) {
  return bfp200_set_error(BFP200_ENOMEM, ex.what());
}
