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
// V^T P^T, so that a group of up to 8 rows needs no padding to 16.  A lane's
// 16 bytes (4 positions x 8 dims, 8 positions x 4 dims) decode into A registers
// without exchange.  Each warp fetches its blocks with cp.async into its own
// ring in shared memory, consecutive lanes consecutive 16 bytes: a lane's own
// units lie 64 bytes apart, and fetched straight to registers every sector
// crossed L2 twice.  S^T's accumulators become P^T's operand by
// one 8x8 transpose (movmatrix) per 8 positions.
//
// Rounding.  K is exact in the operand type; Q is split into as many operands
// of that type as hold all its bits (1 for 16-bit types, 3 bfloat16 for
// 32-bit); V and P use binary16, in which V 2^-4 is exact and P = 2^P_EXP
// exp(s - max) (room for a maximum that is behind) keeps 11 bits (bfloat16
// results: an error of 2^-12 beside the result's own 2^-9), or 22 bits in two
// operands where the result is binary16 or 32-bit.  Scores, maxima, sums and
// accumulators are 32-bit.
//
// What bounds it.  The cache is read once (ncu: 321 MB for 320), but a
// pair of cached values takes 5.3 thread instructions, most of them decoding: at
// 64 sequences of up to 8191 positions, 32 / 8 heads of 128, 57% of the issue
// slots and 53% of the ALU are taken while the cache comes at 3.7 TB/s (86 us; 49
// at the measured copy bandwidth), with 12 warps an SM.  Short or few sequences
// are bound by the chain of one item (lengths, page, first block, joining): 256
// sequences of up to 2047, 9 / 3 heads of 64, take 36 us where the bytes take 10;
// a call for one sequence of 176 takes 14 us, launches included.
//
// Work split.  All (sequence, KV head, row tile) items are laid end to end in
// blocks of 32 positions (64 at heads of 64 and fewer) and cut evenly over the CTAs on the device, from the
// lengths there; cuts near an item's end move onto it.  Cut items leave
// partial sums that a second, dependent launch joins in a fixed order.
#include "kv4_attn.cuh"

#include <cmath>
#include <exception>
#include <string>
#include <type_traits>

int bfp200_set_error(int code, const std::string& msg);   // engine.cu

namespace bfp {
namespace kv4 {
namespace {

// Positions of one step of a warp: 32-position tiles of the tensor-core
// operands, two of them where the head dim leaves room, so that a step's fixed
// work (addresses, waits, the test of the maximum) is shared by more values.
template <int HD> constexpr int SUB = HD <= 64 ? 2 : 1;
template <int HD> constexpr int BLK_OF = 32 * SUB<HD>;
constexpr int MINB = 4;            // blocks that are not worth a second CTA: one for each warp
// An item's fixed cost (its queries, first loads and joining) in blocks, for
// the cuts (256 sequences of up to 2047, 9 / 3 heads of 64: 41.7 us at 0, 36.2 at 4).
constexpr int ITEM = 4;
// ---- the split ---------------------------------------------------------------
struct Seq : Span {
  int blk0, nb, rt;                // first block, blocks plus ITEM, row tiles
};

// Blocks before each sequence (or chunk of `per` sequences, where there are
// more than SCH), summed by every CTA for itself.
constexpr int SCH = 256;
struct Sched {
  long long pre[SCH + 1];
  long long total, geff, delta;
  Span span[SCH];                    // the sequences themselves, where per == 1
  long long wsum[16], wit[16];
  int per;
};

// What follows from a sequence's tokens and positions.
template <int NR, int BLK>
__device__ __forceinline__ Seq seq_make(const AttnArgs& a, const Span& p) {
  Seq r;
  static_cast<Span&>(r) = p;
  const long long first = a.window ? (long long)p.qp0 - a.window + 1 : 0;
  r.blk0 = first > 0 ? min((int)(first / BLK), max(p.len - 1, 0) / BLK) : 0;
  r.nb = max((p.len + BLK - 1) / BLK - r.blk0, 1) + ITEM;
  const long long rows = (long long)p.n_q * a.group;
  r.rt = (int)((rows + NR - 1) / NR);
  return r;
}
template <int NR, int BLK>
__device__ __forceinline__ Seq seq_of(const AttnArgs& a, int s) { return seq_make<NR, BLK>(a, span_of(a.b, s)); }

// Fills the schedule; every thread of the CTA takes part.
template <int NR, int BLK, int THR>
__device__ void make_sched(const AttnArgs& a, Sched& s) {
  constexpr int C = (SCH + THR - 1) / THR;                  // chunks of a thread
  const int per = (a.b.n_seq + SCH - 1) / SCH, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  long long w[C] = {}, sum = 0, items = 0;
  #pragma unroll
  for (int k = 0; k < C; ++k) {
    const int c = threadIdx.x * C + k;
    w[k] = 0;
    if (c >= SCH) break;
    for (int i = c * per; i < min((c + 1) * per, a.b.n_seq); ++i) {
      const Seq q = seq_of<NR, BLK>(a, i);
      if (per == 1) s.span[c] = q;
      const long long n = (long long)q.rt * a.b.H;
      items += n;
      w[k] += n * q.nb;
    }
    sum += w[k];
  }
  long long inc = sum;
  #pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const long long y = __shfl_up_sync(0xffffffffu, inc, o), z = __shfl_xor_sync(0xffffffffu, items, o);
    if (lane >= o) inc += y;
    items += z;
  }
  if (lane == 31) { s.wsum[warp] = inc; s.wit[warp] = items; }
  __syncthreads();
  long long before = 0, total = 0, n_items = 0;
  #pragma unroll
  for (int k = 0; k < THR / 32; ++k) {
    if (k < warp) before += s.wsum[k];
    total += s.wsum[k];
    n_items += s.wit[k];
  }
  long long at = before + inc - sum;
  #pragma unroll
  for (int k = 0; k < C; ++k) {
    if (threadIdx.x * C + k < SCH) s.pre[threadIdx.x * C + k] = at;
    at += w[k];
  }
  if (threadIdx.x == 0) {
    s.pre[SCH] = total;
    s.total = total;
    s.geff = max(min((long long)a.grid, max(n_items, (total + MINB - 1) / MINB)), 1LL);
    s.delta = max(total / (s.geff * 32), (long long)(ITEM + 1));   // no cut leaves less than a block
    s.per = per;
  }
  __syncthreads();
}

struct Item {
  int seq, idx;                    // idx = head * rt + row tile
  long long start, end;            // its blocks
  Seq q;
};

// What a CTA needs again behind an item's loop, in shared memory meanwhile: the
// loop has no registers left (64 sequences of up to 4000 positions, 32 / 8 heads of 64,
// float32: 280 bytes of spills a thread and 55.8 us with it in registers, 8 and 49.3 so).
struct Held {
  Item it;
  long long x, xe, x1;             // the CTA's blocks of the item, the end of its share
  int h, r0, rows;
};

// The item that holds block x (0 <= x < total).
template <int NR, int BLK>
__device__ Item item_at(const AttnArgs& a, const Sched& s, long long x) {
  int lo = 0, hi = SCH;                                     // pre[lo] <= x < pre[hi]
  #pragma unroll 1
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (s.pre[mid] <= x) lo = mid; else hi = mid;
  }
  Item it;
  long long at = s.pre[lo];
  if (s.per == 1) {
    it.seq = lo;
    it.q = seq_make<NR, BLK>(a, s.span[lo]);
  } else {
    it.seq = lo * s.per;
    #pragma unroll 1
    for (;; ++it.seq) {
      it.q = seq_of<NR, BLK>(a, it.seq);
      const long long w = (long long)it.q.rt * a.b.H * it.q.nb;
      if (x < at + w || it.seq + 1 >= a.b.n_seq) break;
      at += w;
    }
  }
  it.idx = (int)div_small(x - at, it.q.nb);
  it.start = at + (long long)it.idx * it.q.nb;
  it.end = it.start + it.q.nb;
  return it;
}

// First block of CTA i: an even share, moved onto an item's edge if one is near.
template <int NR, int BLK>
__device__ long long bound(const AttnArgs& a, const Sched& s, long long i) {
  const long long x = div_small(i * s.total, s.geff);
  if (x <= 0 || x >= s.total) return x <= 0 ? 0 : s.total;
  const Item it = item_at<NR, BLK>(a, s, x);
  const long long before = x - it.start, after = it.end - x;
  if (before <= after) return before <= s.delta ? it.start : x;
  return after <= s.delta ? it.end : x;
}

// A warp's ring of 32-position tiles in shared memory, filled by cp.async with
// consecutive 16-byte units per lane (a lane's own operand bytes lie 64 bytes
// apart: fetched directly, every 32-byte sector would cross L2 twice).  A
// unit's place is its index with low bits exchanged, so that the operand
// reads, 8 lanes at a time, meet 8 different bank groups.
template <int HD>
struct Ring {
  static constexpr int KU = HD / 32;                      // 16-byte units of a lane: keys, and values
  static constexpr int NKE = KU % 2 == 0 ? KU / 2 : KU;   // distinct exponent tiles of the lane's key units
  static constexpr int NVE = KU == 3 ? 3 : 1;             // ... of its value units
  static constexpr int KES = HD == 128 ? 48 : 32, VES = 32;      // bytes between the exponents of two tiles
  static constexpr int KE = HD * 16, KB1 = KE + HD / 16 * KES, VE = HD * 16, VB1 = VE + HD / 16 * VES;
  static constexpr int KB = SUB<HD> * KB1, VB = SUB<HD> * VB1;   // bytes of a stage of keys, of values
  // key unit (quad g, unit t KU + w), value unit (oct t, unit g KU + w)
  __device__ static __forceinline__ int k_place(int u) {
    return HD == 128 ? u ^ (u >> 2 & 3) ^ (u >> 4 & 1) << 2 : HD == 64 ? u ^ (u >> 3 & 1) : u;
  }
  __device__ static __forceinline__ int v_place(int u) {
    return HD == 128 ? u ^ (u >> 5 & 3) : HD == 64 ? u ^ (u >> 4 & 1) ^ (u >> 5 & 1) << 2
         : HD == 32 ? u ^ (u >> 3 & 3) << 1 : u ^ (u / 24 & 3) << 1;
  }
  // place(32 i + lane) * 16 - place(lane) * 16, given an address that holds place(lane) and is a multiple of 128 else
  __device__ static __forceinline__ int k_move(int i, unsigned at) { return i * 512; }
  __device__ static __forceinline__ int v_move(int i, unsigned at) {
    const int x = HD == 128 ? i : HD == 64 ? i << 2 : 0;
    if (HD == 96) {
      const int l = threadIdx.x & 31;
      return (v_place(32 * i + l) - v_place(l)) * 16;
    }
    return i * 512 + (int)((at ^ (x << 4)) - at);
  }
};
// Launch shape by row tiles: warps, CTAs of an SM, stages of a warp's ring.
// CTAs of 4 warps rather than 8: one's start and joining run beside another's
// loop.  Registers set their number: 128 at HD <= 64, 168 above (64 sequences
// of 4608 positions, 32 / 8 heads of 128: 3 x 4 warps 91 us, 2 x 6 98 us, 1 x 12
// 97 us, 2 x 8 at 128 registers 107 us; 37 of 8192, 24 / 8 heads of 64: 4 x 4
// warps 55 us, 3 x 8 at 80 registers 69 us).
template <int HD, int NT> struct Shape {
  static constexpr int W = 4, CTAS = NT == 1 ? (HD <= 64 ? 4 : 3) : NT == 2 && HD <= 64 ? 3 : 2;
  static constexpr int STAGES = HD == 128 || HD == 64 ? 2 : 3;   // of keys; values have one more
  static constexpr int NR = NT * 8;
  static constexpr int RING = W * (STAGES * Ring<HD>::KB + (STAGES + 1) * Ring<HD>::VB), MERGE = W * NR * (HD + 2) * 4;
  template <int QS> static constexpr size_t smem() {
    return (size_t)(HD / 16) * NT * QS * 32 * 8 + (RING > MERGE ? RING : MERGE);
  }
};

template <typename T, int HD, int NT>
__global__ void __launch_bounds__(Shape<HD, NT>::W * 32, Shape<HD, NT>::CTAS) attn_kernel(const AttnArgs a) {
  using SH = Shape<HD, NT>;
  using RG = Ring<HD>;
  constexpr int W = SH::W, STAGES = SH::STAGES, SB = SUB<HD>, BLK = BLK_OF<HD>;
  constexpr int NR = NT * 8, KU = HD / 32, QS = Kind<T>::QS, PS = Kind<T>::PS, REC9 = HD * 9 / 8;
  constexpr bool HALF_K = Kind<T>::HALF_K;
  extern __shared__ __align__(128) unsigned char smem[];
  uint2* s_q = reinterpret_cast<uint2*>(smem);                        // [HD/16][NT][QS][32]
  unsigned char* k_ring = smem + HD / 16 * NT * QS * 32 * 8 + (threadIdx.x >> 5) * (SH::RING / W);
  unsigned char* v_ring = k_ring + STAGES * RG::KB;
  float* s_o = reinterpret_cast<float*>(s_q + HD / 16 * NT * QS * 32);  // after the loop, over the rings: [W][NR][HD]
  float* s_m = s_o + W * NR * HD;                                     // [W][NR], [W][NR]
  float* s_l = s_m + W * NR;
  __shared__ Sched sch;
  __shared__ Held held;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, t = lane & 3;
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  make_sched<NR, BLK, W * 32>(a, sch);
  clear_rows<T, HD>(a, blockIdx.x * W + warp, gridDim.x * W);
  if (tid == 0 && a.cuts) {
    a.cuts[blockIdx.x].parts = 0;
    if (blockIdx.x == 0) a.status->code = BFP200_OK;                    // (no wait here can run out)
  }
  if ((long long)blockIdx.x >= sch.geff || sch.total == 0) return;
  long long x = bound<NR, BLK>(a, sch, (long long)blockIdx.x + (lane & 1));   // both bounds at once
  long long x1 = __shfl_sync(0xffffffffu, x, 1);
  x = __shfl_sync(0xffffffffu, x, 0);
  const int page = a.b.page, rec_bytes = page * REC9;
  const long long page_bytes = (long long)rec_bytes * a.b.H;
  const Magic mg = magic_numbers();
  Item it;
  if (x < x1) it = item_at<NR, BLK>(a, sch, x);
  while (x < x1) {
    long long xe = min(x1, it.end);
    if (xe <= x) break;                                               // lengths changed during the call
    const int rt = it.q.rt;
    int h = it.idx / rt, r0 = (it.idx - h * rt) * NR;
    int rows = min(NR, it.q.n_q * a.group - r0);
    const int len = it.q.len, qp0 = it.q.qp0;
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
      for (int k = 0; k < QS; ++k) s_q[((st * NT + nt) * QS + k) * 32 + l] = make_uint2(o0[k] ^ a.q_flip, o1[k] ^ a.q_flip);
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
    float m[NT][2], ref[NT][2], lsum[NT][2], O[KU][2][NT][4];
    #pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      m[nt][0] = m[nt][1] = -INFINITY;
      ref[nt][0] = ref[nt][1] = 0.f;
      lsum[nt][0] = lsum[nt][1] = 0.f;
      #pragma unroll
      for (int w = 0; w < KU; ++w)
        #pragma unroll
        for (int n = 0; n < 2; ++n)
          #pragma unroll
          for (int k = 0; k < 4; ++k) O[w][n][nt][k] = 0.f;
    }
    if (tid == 0) held = Held{it, x, xe, x1, h, r0, rows};
    __syncthreads();

    // this segment's blocks that some row sees, as positions
    const int skip = x == it.start ? 0 : (int)(x - it.start) - ITEM;   // blocks of CTAs before this one
    const int first = max(skip + it.q.blk0, any_lo / BLK);
    const int last = min((int)(xe - it.start) - ITEM + it.q.blk0, (any_hi + BLK - 1) / BLK);
    const int* bt = a.b.bt + (long long)it.seq * a.b.bt_ld;
    const auto page_at = [&](int pos) -> int {
      const int i = pos >> a.b.page_shift;
      return i < a.b.max_pages ? __ldg(bt + i) : -1;
    };
    const uint8_t* pool_h = a.b.pool + (long long)h * rec_bytes;
    const bool one_page = page >= BLK;                                // a block lies in one page
    const bool halves = page < 32;                                    // a tile's 32 positions lie in two pages
    int pk[2 * SB];                                                   // pages of the next block to fetch
    const auto pages = [&](int base) {
      pk[0] = page_at(base);
      if (!one_page) {
        #pragma unroll
        for (int i = 1; i < 2 * SB; ++i) pk[i] = halves || i % 2 == 0 ? page_at(base + 16 * i) : pk[i - 1];
      }
    };
    const unsigned k_dst = su32(k_ring) + RG::k_place(lane) * 16, v_dst = su32(v_ring) + RG::v_place(lane) * 16;
    const unsigned e_dst = lane < HD / 8 ? su32(k_ring) + RG::KE + (lane >> 1) * RG::KES + (lane & 1) * 16
                                         : su32(v_ring) + RG::VE + ((lane >> 1) - HD / 16) * RG::VES + (lane & 1) * 16;
    const int e_stage = lane < HD / 8 ? RG::KB1 : RG::VB1, e_src = page * HD + (lane >> 1) * page + (lane & 1) * 16 - lane * 16;
    const auto load = [&](int ks, int vs, int base) {
      if (one_page && (unsigned)pk[0] < (unsigned)a.b.n_pages) {
        const uint8_t* src = pool_h + (long long)pk[0] * page_bytes + (base & (page - 1)) * (HD / 2) + lane * 16;
        const uint8_t *vsrc = src + page * HD / 2, *esrc = src + (e_src - (base & (page - 1)) * (HD / 2 - 1));
        const unsigned kd = k_dst + ks * RG::KB, vd = v_dst + vs * RG::VB, ed = e_dst + (lane < HD / 8 ? ks : vs) * SB * e_stage;
        #pragma unroll
        for (int sub = 0; sub < SB; ++sub) {                          // 32 positions on: 16 HD bytes of keys and of values
          #pragma unroll
          for (int i = 0; i < KU; ++i) {
            cp16(kd + sub * RG::KB1 + RG::k_move(i, kd), src + sub * 16 * HD + i * 512);
            cp16(vd + sub * RG::VB1 + RG::v_move(i, vd), vsrc + sub * 16 * HD + i * 512);
          }
          if (lane < HD / 4) cp16(ed + sub * e_stage, esrc + sub * 32);   // 32 bytes of every key and value tile
        }
        return;
      }
      #pragma unroll 1
      for (int i = 0; i < 2 * SB; ++i) {                              // 16 positions at a time; of no page: zeros
        unsigned char *kst = k_ring + ks * RG::KB + (i >> 1) * RG::KB1, *vst = v_ring + vs * RG::VB + (i >> 1) * RG::VB1;
        const int hf = i & 1, at = (base + 16 * i) & (page - 1);
        int pg = pk[0];
        #pragma unroll
        for (int k = 1; k < 2 * SB; ++k) pg = !one_page && i == k ? pk[k] : pg;
        const bool ok = (unsigned)pg < (unsigned)a.b.n_pages;
        const uint8_t* rec = pool_h + (ok ? (long long)pg * page_bytes : 0);
        const uint4 zero = make_uint4(0x88888888u, 0x88888888u, 0x88888888u, 0x88888888u);
        #pragma unroll
        for (int u0 = 0; u0 < HD / 2; u0 += 32) {
          const int u = u0 + lane;
          if (u < HD / 2) {
            unsigned char *kd = kst + RG::k_place(u + hf * (HD / 2)) * 16, *vd = vst + RG::v_place(u + hf * (HD / 2)) * 16;
            const uint8_t* from = rec + at * (HD / 2) + u * 16;
            if (ok) {
              cp16(su32(kd), from);
              cp16(su32(vd), from + page * HD / 2);
            } else {
              *reinterpret_cast<uint4*>(kd) = zero;
              *reinterpret_cast<uint4*>(vd) = zero;
            }
          }
        }
        if (lane < HD / 8) {
          unsigned char* d = (lane < HD / 16 ? kst + RG::KE + lane * RG::KES : vst + RG::VE + (lane - HD / 16) * RG::VES) + hf * 16;
          if (ok) cp16(su32(d), rec + page * HD + lane * page + at);
          else *reinterpret_cast<uint4*>(d) = make_uint4(0x01010101u, 0x01010101u, 0x01010101u, 0x01010101u);
        }
      }
    };

    // S^T = K Q^T: tiles of rows (position 4 g, 4 g + 1) and (4 g + 2, 4 g + 3).
    // (The query's low parts are summed apart: the tensor core cuts addends off at the sum's last bit.)
    float S[SB * 2][NT][4], S_low[QS > 1 ? SB * 2 : 1][QS > 1 ? NT : 1][4];
    unsigned P[PS][SB * 4][NT];
    const auto scores = [&](int ks) {
      const unsigned char* st = k_ring + ks * RG::KB;
      #pragma unroll
      for (int i = 0; i < SB * 2; ++i)
        #pragma unroll
        for (int nt = 0; nt < NT; ++nt)
          #pragma unroll
          for (int k = 0; k < 4; ++k) {
            S[i][nt][k] = 0.f;
            if constexpr (QS > 1) S_low[i][nt][k] = 0.f;
          }
      constexpr int WPT = RG::NKE == KU ? 1 : 2;                  // units of one exponent tile
      #pragma unroll
      for (int sub = 0; sub < SB; ++sub) {
        #pragma unroll
        for (int e = 0; e < RG::NKE; ++e) {
          const unsigned eb = *reinterpret_cast<const unsigned*>(st + sub * RG::KB1 + RG::KE + (WPT == 1 ? (t * KU + e) / 2 : t * RG::NKE + e) * RG::KES + 4 * g);
          KeyScaleT<HALF_K> sc[4];
          #pragma unroll
          for (int i = 0; i < 4; ++i) sc[i] = key_scale<HALF_K>(prmt(eb, 0u, i | 0x40 | i << 8 | 0x4000));
          #pragma unroll
          for (int w2 = 0; w2 < WPT; ++w2) {
            const int w = e * WPT + w2;
            const uint4 kv = *reinterpret_cast<const uint4*>(st + sub * RG::KB1 + RG::k_place(g * (HD / 8) + t * KU + w) * 16);
            const unsigned word[4] = {kv.x, kv.y, kv.z, kv.w};
            unsigned op[4][4];                                       // [position][pair]
            #pragma unroll
            for (int i = 0; i < 4; ++i) key_pairs<HALF_K>(mg, word[i], sc[i], op[i]);
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
                    if constexpr (HALF_K) mma_f16(S[sub * 2 + i][nt], fr, qb);
                    else if (k == 0) mma_bf16(S[sub * 2 + i][nt], fr, qb);
                    else mma_bf16(S_low[QS > 1 ? sub * 2 + i : 0][QS > 1 ? nt : 0], fr, qb);
                  }
                }
          }
        }
      }
    };
    // Running softmax, S^T to P^T.  The reference m of a row moves only when a score
    // passes it by more than `slack` (in powers of two; P stays below 2^16).
    const auto weights = [&](int base, bool whole) {
      float top[NT][2];
      bool passed = false;
      #pragma unroll
      for (int nt = 0; nt < NT; ++nt)
        #pragma unroll
        for (int c = 0; c < 2; ++c) {
          #pragma unroll
          for (int i = 0; i < SB * 4; ++i) {
            float& s = S[i >> 1][nt][(i & 1) * 2 + c];
            if constexpr (QS > 1) s += S_low[i >> 1][nt][(i & 1) * 2 + c];
            if (!whole) {
              const int p = base + (i >> 2) * 32 + 4 * g + (i & 3);
              s = p < hi[nt][c] && p >= lo[nt][c] ? s : -INFINITY;
            }
          }
          top[nt][c] = fmaxf(fmaxf(S[0][nt][c], S[0][nt][2 + c]), fmaxf(S[1][nt][c], S[1][nt][2 + c]));
          if constexpr (SB > 1)
            top[nt][c] = fmaxf(top[nt][c], fmaxf(fmaxf(S[2][nt][c], S[2][nt][2 + c]), fmaxf(S[3][nt][c], S[3][nt][2 + c])));
          passed |= top[nt][c] > m[nt][c] + a.slack[PS - 1];
        }
      if (__any_sync(0xffffffffu, passed)) {
        #pragma unroll
        for (int nt = 0; nt < NT; ++nt)
          #pragma unroll
          for (int c = 0; c < 2; ++c) {
            #pragma unroll
            for (int o = 4; o < 32; o <<= 1) top[nt][c] = fmaxf(top[nt][c], __shfl_xor_sync(0xffffffffu, top[nt][c], o));
            const float mn = fmaxf(m[nt][c], top[nt][c]);
            const float al = mn == -INFINITY ? 1.f : ex2((m[nt][c] - mn) * a.scale_log2);
            m[nt][c] = mn;
            ref[nt][c] = mn == -INFINITY ? 0.f : mn * a.scale_log2 - P_EXP<PS>;
            lsum[nt][c] *= al;
            #pragma unroll
            for (int w = 0; w < KU; ++w)
              #pragma unroll
              for (int n = 0; n < 2; ++n) {
                O[w][n][nt][c] *= al;
                O[w][n][nt][2 + c] *= al;
              }
          }
      }
      #pragma unroll
      for (int nt = 0; nt < NT; ++nt)
        #pragma unroll
        for (int i = 0; i < SB * 4; ++i) {
          const float p0 = ex2(__fmaf_rn(S[i >> 1][nt][(i & 1) * 2], a.scale_log2, -ref[nt][0]));
          const float p1 = ex2(__fmaf_rn(S[i >> 1][nt][(i & 1) * 2 + 1], a.scale_log2, -ref[nt][1]));
          lsum[nt][0] += p0;
          lsum[nt][1] += p1;
          const __half2 hp = __floats2half2_rn(p0, p1);
          P[0][i][nt] = transpose8(as_u(hp));
          if constexpr (PS == 2) {
            const float2 back = __half22float2(hp);
            P[1][i][nt] = transpose8(as_u(__floats2half2_rn(p0 - back.x, p1 - back.y)));
          }
        }
    };
    // O^T += V^T P^T
    const auto accumulate = [&](int vs) {
      #pragma unroll
      for (int sub = 0; sub < SB; ++sub) {
        const unsigned char* st = v_ring + vs * RG::VB + sub * RG::VB1;
        ScaleH sc[4];
        #pragma unroll
        for (int w = 0; w < KU; ++w) {
          if (w == 0 || RG::NVE > 1) {
            const uint2 eb = *reinterpret_cast<const uint2*>(st + RG::VE + (g * KU + w) / 4 * RG::VES + 8 * t);
            #pragma unroll
            for (int i = 0; i < 4; ++i)                              // positions 8 t + i and 8 t + i + 4
              sc[i] = scale_h(prmt(eb.x, eb.y, i * 0x0101 | 0x0080 | (4 + i) << 8 | (12 + i) << 12));
          }
          const uint4 vv = *reinterpret_cast<const uint4*>(st + RG::v_place(t * (HD / 4) + g * KU + w) * 16);
          const unsigned word[4] = {vv.x, vv.y, vv.z, vv.w};
          #pragma unroll
          for (int j = 0; j < 2; ++j) {
            unsigned op[2][4];                                     // [pair of positions][dim]
            pairs_h(mg, word[2 * j], sc[2 * j], op[0]);
            pairs_h(mg, word[2 * j + 1], sc[2 * j + 1], op[1]);
            #pragma unroll
            for (int n = 0; n < 2; ++n) {
              const unsigned fr[4] = {op[0][2 * n], op[0][2 * n + 1], op[1][2 * n], op[1][2 * n + 1]};
              #pragma unroll
              for (int nt = 0; nt < NT; ++nt)
                #pragma unroll
                for (int k = 0; k < PS; ++k)
                  mma_f16(O[w][n][nt], fr, make_uint2(P[k][sub * 4 + 2 * j][nt], P[k][sub * 4 + 2 * j + 1][nt]));
            }
          }
        }
      }
    };
    // Bytes at positions that no row sees may be anything; exponent 0 makes
    // their values 0 (and never NaN, which a weight of 0 would not remove).
    const int v_hi = min(len, any_hi);
    const auto clear = [&](int vs, int base) {
      #pragma unroll
      for (int sub = 0; sub < SB; ++sub) {
        const int p = base + 32 * sub + lane;
        if (p >= v_hi || p < any_lo)
          for (int tile = 0; tile < HD / 16; ++tile) v_ring[vs * RG::VB + sub * RG::VB1 + RG::VE + tile * RG::VES + lane] = 0;
      }
      __syncwarp();
    };

    // The scores of a block are computed beside the accumulation of the one
    // before: two independent chains for the scheduler.
    if (first + warp < last) {
      int blk = first + warp, ahead = blk;
      pages(blk * BLK);
      const auto fetch = [&](int ks, int vs) {                        // the block `ahead`, and the next one's pages
        __syncwarp();
        if (ahead < last) {
          load(ks, vs, ahead * BLK);
          ahead += W;
          if (ahead < last) pages(ahead * BLK);
        }
        asm volatile("cp.async.commit_group;" ::: "memory");
      };
      #pragma unroll
      for (int i = 0; i < STAGES; ++i) fetch(i, i);
      int ks = 0, vs = 0;
      const auto arrive = [&]() {                                     // block blk is here; is it whole?
        asm volatile("cp.async.wait_group %0;" :: "n"(STAGES - 1) : "memory");
        __syncwarp();
        const int base = blk * BLK;
        const bool whole = base + BLK <= all_hi && base >= all_lo;
        if (!whole) clear(vs, base);
        return whole;
      };
      bool whole = arrive();
      scores(ks);
      weights(blk * BLK, whole);
      fetch(ks, STAGES);
      for (;;) {
        const int before = vs;
        blk += W;
        if (blk >= last) break;
        ks = ks + 1 == STAGES ? 0 : ks + 1;
        vs = vs == STAGES ? 0 : vs + 1;
        whole = arrive();
        scores(ks);
        accumulate(before);
        weights(blk * BLK, whole);
        fetch(ks, before);
      }
      accumulate(vs);
    }
    __syncthreads();                                                  // the rings become the joining buffers
    it = held.it;
    x = held.x; xe = held.xe; x1 = held.x1;
    h = held.h; r0 = held.r0; rows = held.rows;

    // ---- join the warps
    #pragma unroll
    for (int nt = 0; nt < NT; ++nt)
      #pragma unroll
      for (int c = 0; c < 2; ++c) {
        #pragma unroll
        for (int o = 4; o < 32; o <<= 1) lsum[nt][c] += __shfl_xor_sync(0xffffffffu, lsum[nt][c], o);
        const int r = nt * 8 + 2 * t + c;
        if (g == 0) { s_m[warp * NR + r] = m[nt][c] * a.scale_log2; s_l[warp * NR + r] = lsum[nt][c]; }
        #pragma unroll
        for (int w = 0; w < KU; ++w)
          #pragma unroll
          for (int n = 0; n < 2; ++n)
            *reinterpret_cast<float2*>(s_o + (warp * NR + r) * HD + (g * KU + w) * 4 + 2 * n) =
                make_float2(O[w][n][nt][c], O[w][n][nt][2 + c]);
      }
    __syncthreads();
    const bool full = x == it.start && xe == it.end;
    if (x == it.start && xe < it.end && tid == 0) {
      // the parts end at the last boundary below the item's end, unless that was moved onto it
      const long long c = blockIdx.x;
      long long e = min(sch.geff, div_small(it.end * sch.geff + sch.total - 1, sch.total));
      while (e - 1 > c + 1 && bound<NR, BLK>(a, sch, e - 1) >= it.end) --e;
      a.cuts[c] = Cut{(int)(e - c), it.q.q0, rows, r0, h * a.group, 0, {0, 0}};
    }
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
        if (d == 0 && a.lse) a.lse[(long long)(it.q.q0 + j) * a.HQ + head] = L == 0.f ? -INFINITY : (M + log2f(L) - P_EXP<PS>) * LN2;
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
        it = item_at<NR, BLK>(a, sch, x);
      }
    }
  }
}

// Items of at most MINB blocks are never cut: an edge lies within ITEM + 1 of
// every place in them.  No workspace then, and no joining launch.
template <int HD> bool never_cut(const Batch& b) { return (long long)b.max_pages * b.page <= MINB * BLK_OF<HD>; }
static_assert(MINB + ITEM <= 2 * (ITEM + 1), "items of MINB blocks stay whole");

template <typename T, int HD, int NT>
cudaError_t launch_attn(AttnArgs a, int n_sm, void* ws, cudaStream_t s) {
  using SH = Shape<HD, NT>;
  constexpr int W = SH::W, NR = NT * 8;
  constexpr size_t smem = SH::template smem<Kind<T>::QS>();
  static_assert(smem + 2048 <= 227 * 1024, "shared memory");
  auto* kern = attn_kernel<T, HD, NT>;
  static std::atomic<unsigned char> allowed[128];
  cudaError_t e = allow_smem(kern, smem, allowed);
  if (e != cudaSuccess) return e;
  a.grid = n_sm * SH::CTAS;
  const bool whole = a.b.n_seq == 0 || never_cut<HD>(a.b);
  a.status = whole ? nullptr : static_cast<Status*>(ws);
  a.cuts = whole ? nullptr : reinterpret_cast<Cut*>(a.status + 1);
  a.part = whole ? nullptr : reinterpret_cast<float*>(a.cuts + a.grid);
  kern<<<a.grid, W * 32, smem, s>>>(a);
  e = cudaGetLastError();
  if (e != cudaSuccess) return e;
  if (whole) return cudaSuccess;
  return launch_join<T, HD, NR, false>(a, 4, s);
}

// Row tile of a call, by the sequences' average of tokens times the group; 8
// stands for the prompt kernel.  At heads of 128 it is ahead from 64 rows on (16
// sequences of up to 4000 positions, 24 tokens of 32 / 8 heads: 82 us against 123),
// at 64 and fewer dims, where decoding is half and the softmax all of the work,
// from some 300 (100 tokens of 9 / 3 heads: 90 against 96; 48 tokens: 66 against 57).
// Heads of 96 go with 128 and 32 with 64, unmeasured.
// 32-bit queries would not fit its shared memory.
int pick_nt(const Batch& b, int group, int hd, bool wide) {
  if (b.n_seq == 0) return 1;
  const long long rows = ((long long)b.T + b.n_seq - 1) / b.n_seq * group;
  return rows <= 8 ? 1 : rows <= 16 ? 2 : wide || rows <= (hd > 64 ? 32 : 256) ? 4 : 8;
}
// Room for the partial sums of any call with this head dim; none where nothing is cut.
size_t ws_bytes(const Batch& b, int hd, int nt, int n_sm) {
  if (b.n_seq == 0) return 0;
  if (nt != 8 && (hd > 64 ? never_cut<128>(b) : never_cut<64>(b))) return 0;
  size_t most = 0;
  for (int nt = 1; nt <= 4; nt *= 2) {
    const size_t grid = (size_t)n_sm * 4, b = sizeof(Status) + grid * (sizeof(Cut) + 2 * nt * 8 * (hd + 2) * 4);
    most = b > most ? b : most;
  }
  const size_t p = prompt_ws_bytes(hd, n_sm);
  return p > most ? p : most;
}

template <typename T, int HD>
cudaError_t by_nt(const AttnArgs& a, int nt, int n_sm, int spin, void* ws, cudaStream_t s) {
  if constexpr (!std::is_same<T, float>::value)
    if (nt == 8) return launch_prompt<T, HD>(a, n_sm, spin, ws, s);
  return nt == 1 ? launch_attn<T, HD, 1>(a, n_sm, ws, s)
       : nt == 2 ? launch_attn<T, HD, 2>(a, n_sm, ws, s)
                 : launch_attn<T, HD, 4>(a, n_sm, ws, s);
}
template <typename T>
cudaError_t by_hd(int hd, const AttnArgs& a, int nt, int n_sm, int spin, void* ws, cudaStream_t s) {
  return hd == 32 ? by_nt<T, 32>(a, nt, n_sm, spin, ws, s)
       : hd == 64 ? by_nt<T, 64>(a, nt, n_sm, spin, ws, s)
       : hd == 96 ? by_nt<T, 96>(a, nt, n_sm, spin, ws, s)
                  : by_nt<T, 128>(a, nt, n_sm, spin, ws, s);
}

// What is wrong with a call's query heads, or null.  The kernels count the rows
// of a KV head, and the items of a sequence, in 32 bits.
const char* bad_heads(const Batch& b, long long HQ) {
  if (HQ < 1 || HQ > (1LL << 16) || HQ % b.H) return "H_Q must be a positive multiple of H_KV";
  if (b.T * (HQ / b.H) > (1LL << 31) - 512 || b.T * HQ > (1LL << 33)) return "too many rows (tokens times query heads)";
  return nullptr;
}

// probe: a call of the prompts' kernel, whose waits give up at once
int attention(const char* who, const bfp200_kv4_attention_args* in, bool probe, void* stream) {
  const auto bad = [&](const char* what) { return bfp200_set_error(BFP200_EINVAL, std::string(who) + ": " + what); };
  if (!in) return bad("no arguments");
  const bfp200_kv4_attention_args& r = *in;
  AttnArgs a;
  if (int rc = fill_batch(r.batch, &a.b, who)) return rc;
  const int es = r.dtype == BFP200_F32 ? 4 : r.dtype == BFP200_F16 || r.dtype == BFP200_BF16 ? 2 : 0;
  if (!es) return bad("dtype must be BFP200_F32, BFP200_F16 or BFP200_BF16");
  if (const char* what = bad_heads(a.b, r.H_Q)) return bad(what);
  if (r.window < 0) return bad("window must not be negative");
  if (!(r.scale - r.scale == 0.0)) return bad("scale must be finite");
  if (a.b.T == 0) return BFP200_OK;
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
  a.window = r.window < (1LL << 31) ? r.window : 1LL << 31;   // (hides nothing; what the kernels add to it stays in range)
  const double sl = std::fabs(r.scale) * 1.4426950408889634 * (r.dtype == BFP200_F16 ? 16.0 : 1.0);   // K is held times 2^-4 there
  if (sl > 1e30) return bad("scale is too large");
  a.scale_log2 = (float)std::fmax(sl, 1e-30);
  a.slack[0] = SLACK<1> / a.scale_log2;
  a.slack[1] = SLACK<2> / a.scale_log2;
  a.q_flip = r.scale < 0 ? 0x80008000u : 0u;
  a.grid = 0;
  a.part = nullptr;
  const int hd = (int)r.batch.HD, nt = pick_nt(a.b, a.group, hd, r.dtype == BFP200_F32);
  if (probe && nt != 8) return bad("not a call of the prompts' kernel");
  const int spin = probe ? 0 : SPIN;
  const size_t need = ws_bytes(a.b, hd, nt, n_sm);
  if (need && (!r.workspace_dev || r.workspace_bytes < (long long)need))
    return bad("the workspace is smaller than bfp200_kv4_attention_workspace says");
  void* const ws = r.workspace_dev;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const cudaError_t e = r.dtype == BFP200_F32 ? by_hd<float>(hd, a, nt, n_sm, spin, ws, s)
                      : r.dtype == BFP200_F16 ? by_hd<__half>(hd, a, nt, n_sm, spin, ws, s)
                                              : by_hd<__nv_bfloat16>(hd, a, nt, n_sm, spin, ws, s);
  if (e != cudaSuccess) return bfp200_set_error(BFP200_ECUDA, std::string(who) + ": " + cudaGetErrorString(e));
  return BFP200_OK;
}

}  // namespace
}  // namespace kv4
}  // namespace bfp

using namespace bfp::kv4;

extern "C" int bfp200_kv4_attention_workspace(const bfp200_kv4_attention_args* in, size_t* bytes) try {
  const char* who = "kv4_attention_workspace";
  const auto bad = [&](const char* what) { return bfp200_set_error(BFP200_EINVAL, std::string(who) + ": " + what); };
  if (!in || !bytes) return bad("no arguments");
  Batch b;
  if (int rc = fill_batch(in->batch, &b, who)) return rc;
  if (const char* what = bad_heads(b, in->H_Q)) return bad(what);
  int n_sm = 0;
  if (int rc = device_ready(who, &n_sm)) return rc;
  const int hd = (int)in->batch.HD;
  *bytes = b.T == 0 ? 0 : ws_bytes(b, hd, pick_nt(b, (int)in->H_Q / b.H, hd, in->dtype == BFP200_F32), n_sm);
  return BFP200_OK;
} catch (const std::exception& ex) {
  return bfp200_set_error(BFP200_ENOMEM, ex.what());
}

extern "C" int bfp200_kv4_attention_dev(const bfp200_kv4_attention_args* in, void* stream) try {
  return attention("kv4_attention_dev", in, false, stream);
} catch (const std::exception& ex) {
  return bfp200_set_error(BFP200_ENOMEM, ex.what());
}

extern "C" int bfp200_kv4_wait_probe(const bfp200_kv4_attention_args* in, void* stream) try {
  return attention("kv4_wait_probe", in, true, stream);
} catch (const std::exception& ex) {
  return bfp200_set_error(BFP200_ENOMEM, ex.what());
}

extern "C" int bfp200_kv4_attention_status(const void* workspace_dev, void* stream) try {
  const char* who = "kv4_attention_status";
  if (reinterpret_cast<uintptr_t>(workspace_dev) % 16) return bfp200_set_error(BFP200_EINVAL, std::string(who) + ": misaligned pointer");
  int n_sm = 0, code = BFP200_OK;
  if (int rc = device_ready(who, &n_sm)) return rc;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  cudaError_t e = workspace_dev ? cudaMemcpyAsync(&code, workspace_dev, sizeof(code), cudaMemcpyDeviceToHost, s) : cudaSuccess;
  if (e == cudaSuccess) e = cudaStreamSynchronize(s);
  if (e != cudaSuccess) return bfp200_set_error(BFP200_ECUDA, std::string(who) + ": " + cudaGetErrorString(e));
  return code == BFP200_OK ? BFP200_OK : bfp200_set_error(BFP200_ETIMEOUT, std::string(who) + ": a bounded device wait timed out");
} catch (const std::exception& ex) {
  return bfp200_set_error(BFP200_ENOMEM, ex.what());
}
