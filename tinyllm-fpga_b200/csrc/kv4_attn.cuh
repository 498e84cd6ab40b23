// kv4_attn.cuh -- what the two attention kernels over the 4-bit cache share:
// arguments, the operands made of cached bytes, and the launch that joins the
// partial sums of items cut over CTAs.  Included by one kernel file each.
#pragma once
#include "kv4.cuh"

#include <cstring>
#include <type_traits>

namespace bfp {
namespace kv4 {

constexpr float LN2 = 0.6931471805599453f;
// P is held times 2^P_EXP, at most 2^(P_EXP + SLACK) = 2^15: with one binary16
// operand it turns subnormal (errors of 2^-32 of the maximum's weight) below
// 2^-21, with two below 2^-28.
template <int PS> constexpr float P_EXP = PS == 1 ? 7.f : 14.f;
template <int PS> constexpr float SLACK = PS == 1 ? 8.f : 1.f;
constexpr float V_UP = 16.f;       // V is held times 2^-4

// An item cut over CTAs c .. c + parts - 1, left by CTA c for the joining launch.
struct Cut {
  int parts;                       // 0: none
  int q0, rows, r0, head0;         // first token, rows, first row, first query head
  int late;                        // a wait of the CTA ran out
  int pad[2];
};

// The workspace: the call's status, a Cut a CTA, partial sums.
struct Status {
  int code;                        // BFP200_OK or BFP200_ETIMEOUT
  int pad[31];                     // (a line: what follows keeps its alignment)
};

struct AttnArgs {
  Batch b;
  const void* q;
  void* out;
  float* lse;                      // [T][HQ] or null
  float* part;                     // partial sums: [CTA][2][NR][HD + 2]
  Cut* cuts;                       // [CTA]: the item that the CTA begins and does not end
  Status* status;
  long long q_ts, q_hs, o_ts, o_hs;
  int HQ, group, causal;
  long long window;                // 0: none
  float scale_log2;                // > 0: a negative scale negates the queries
  float slack[2];                  // SLACK<1>, SLACK<2> in units of the scores
  unsigned q_flip;                 // sign bits to flip in a pair of 16-bit queries
  int grid;                        // CTAs of the first launch
};

// A sequence as the call describes it.  The last token before q_start[s + 1] is at
// position lens[s] - 1, as for append and read: tokens keep their positions where
// the table holds fewer than lens[s] (or the call fewer rows than q_start says).
struct Span { int q0, n_q, len, qp0; };   // first token, tokens, positions that the table holds, position of the first token
__device__ __forceinline__ Span span_of(const Batch& b, int s) {
  const int end = __ldg(b.q_start + s + 1), len = max(__ldg(b.lens + s), 0);
  Span r;
  r.q0 = min(max(__ldg(b.q_start + s), 0), b.T);
  r.n_q = min(max(end, r.q0), b.T) - r.q0;
  r.len = min(len, b.max_pages << b.page_shift);
  r.qp0 = len - (max(end, r.q0) - r.q0);
  return r;
}

// Rows of no sequence, before q_start[0] and from q_start[n_seq] on: zeros and
// -infinity, a row a warp.  Where every row belongs to a sequence it costs two
// loads.
template <typename T, int HD>
__device__ __forceinline__ void clear_rows(const AttnArgs& a, int warp, int warps) {
  const int lead = a.b.n_seq ? min(max(__ldg(a.b.q_start), 0), a.b.T) : 0;
  const int tail = a.b.n_seq ? min(max(__ldg(a.b.q_start + a.b.n_seq), lead), a.b.T) : 0;
  #pragma unroll 1
  for (int t = warp < lead ? warp : tail + warp - lead; t < a.b.T; t = t + warps < lead || t >= tail ? t + warps : t + warps - lead + tail) {
    #pragma unroll 1
    for (int i = threadIdx.x & 31; i < a.HQ * HD; i += 32)
      static_cast<T*>(a.out)[t * a.o_ts + i / HD * a.o_hs + i % HD] = from_f<T>(0.f);
    if (a.lse)
      for (int i = threadIdx.x & 31; i < a.HQ; i += 32) a.lse[(long long)t * a.HQ + i] = -INFINITY;
  }
}

// ---- arithmetic ------------------------------------------------------------------
__device__ __forceinline__ void mma_bf16(float (&c)[4], const unsigned (&a)[4], uint2 b) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
               : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
               : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b.x), "r"(b.y));
}
__device__ __forceinline__ void mma_f16(float (&c)[4], const unsigned (&a)[4], uint2 b) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
               : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
               : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b.x), "r"(b.y));
}
__device__ __forceinline__ unsigned transpose8(unsigned x) {
  unsigned y;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
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
// (x & MASK) | magic in one instruction, which takes one immediate: the magic
// numbers stay in registers.
struct Magic { unsigned h1024, h64, b128; };
__device__ __forceinline__ Magic magic_numbers() {
  Magic m;
  asm volatile("mov.u32 %0, 0x64006400;" : "=r"(m.h1024));
  asm volatile("mov.u32 %0, 0x54005400;" : "=r"(m.h64));
  asm volatile("mov.u32 %0, 0x43004300;" : "=r"(m.b128));
  return m;
}
template <unsigned MASK>
__device__ __forceinline__ unsigned and_or(unsigned x, unsigned magic) {
  unsigned y;
  asm("lop3.b32 %0, %1, %2, %3, 0xEA;" : "=r"(y) : "r"(x), "n"(MASK), "r"(magic));
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
__device__ __forceinline__ void pairs_h(const Magic& mg, unsigned w, const ScaleH& sc, unsigned (&o)[4]) {
  const unsigned w8 = w >> 8;
  const __half2 s = as_h2(sc.s), c0 = as_h2(sc.c1024), c1 = as_h2(sc.c64);
  o[0] = as_u(__hfma2(as_h2(and_or<0x000F000Fu>(w, mg.h1024)), s, c0));
  o[1] = as_u(__hfma2(as_h2(and_or<0x00F000F0u>(w, mg.h64)), s, c1));
  o[2] = as_u(__hfma2(as_h2(and_or<0x000F000Fu>(w8, mg.h1024)), s, c0));
  o[3] = as_u(__hfma2(as_h2(and_or<0x00F000F0u>(w8, mg.h64)), s, c1));
}
// Bfloat16 pairs: 128 + nibble, less 136, scaled; exact.
struct ScaleB { unsigned s, c; };
__device__ __forceinline__ ScaleB scale_b(unsigned bytes) {
  ScaleB r;
  r.s = bytes * 128u + 0x35003500u;                                 // 2^(B - 21)
  r.c = as_u(__hmul2(as_b2(r.s), __floats2bfloat162_rn(-136.f, -136.f)));
  return r;
}
__device__ __forceinline__ void pairs_b(const Magic& mg, unsigned w, const ScaleB& sc, unsigned (&o)[4]) {
  #pragma unroll
  for (int n = 0; n < 4; ++n) o[n] = as_u(__hfma2(as_b2(and_or<0x000F000Fu>(w >> (4 * n), mg.b128)), as_b2(sc.s), as_b2(sc.c)));
}
template <bool HALF> using KeyScaleT = std::conditional_t<HALF, ScaleH, ScaleB>;
template <bool HALF> __device__ __forceinline__ KeyScaleT<HALF> key_scale(unsigned bytes) {
  if constexpr (HALF) return scale_h(bytes);
  else return scale_b(bytes);
}
template <bool HALF> __device__ __forceinline__ void key_pairs(const Magic& mg, unsigned w, const KeyScaleT<HALF>& sc, unsigned (&o)[4]) {
  if constexpr (HALF) pairs_h(mg, w, sc, o);
  else pairs_b(mg, w, sc, o);
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

__device__ __forceinline__ long long div_small(long long x, long long y) {   // 32-bit where it fits: a third of the time
  return ((x | y) >> 32) == 0 ? (long long)((unsigned)x / (unsigned)y) : x / y;
}

__device__ __forceinline__ unsigned su32(const void* p) { return (unsigned)__cvta_generic_to_shared(p); }
__device__ __forceinline__ void cp16(unsigned d, const void* g) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" :: "r"(d), "l"(g) : "memory");
}

namespace {

// Joins the partial sums of the item that CTA blockIdx.x began and others
// ended, part after part in their order.  Behind the prompts' kernel it also
// clears the rows of no sequence, beside that kernel's end, and its last CTA,
// which can have begun no item, gathers the call's status.
template <typename T, int HD, int NR, bool PROMPT>
__global__ void __launch_bounds__(256) join_kernel(const AttnArgs a) {
  constexpr int Q = HD / 4, NG = 256 / Q;          // NG groups of threads share the parts
  __shared__ float4 s_o[NG][Q];
  __shared__ float s_m[NG], s_l[NG];
  if (PROMPT) clear_rows<T, HD>(a, (blockIdx.y * gridDim.x + blockIdx.x) * 8 + threadIdx.x / 32, gridDim.x * gridDim.y * 8);
  asm volatile("griddepcontrol.wait;" ::: "memory");
  if (PROMPT && blockIdx.x + 1 == gridDim.x && blockIdx.y == 0) {
    int late = 0;
    for (int c = threadIdx.x; c < a.grid; c += 256) late |= __ldcg(&a.cuts[c].late);
    late = __syncthreads_or(late);
    if (threadIdx.x == 0) a.status->code = late ? BFP200_ETIMEOUT : BFP200_OK;
  }
  const int4 c0 = __ldcg(reinterpret_cast<const int4*>(a.cuts + blockIdx.x));
  const int n = c0.x, rows = c0.z;
  if (n == 0) return;
  const int head0 = __ldcg(&a.cuts[blockIdx.x].head0);
  const int grp = threadIdx.x / Q, d4 = threadIdx.x % Q;
  for (int r = blockIdx.y; r < rows; r += gridDim.y) {
    float M = -INFINITY, L = 0.f;
    float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
    if (grp < NG) {
      #pragma unroll 4
      for (int k = grp; k < n; k += NG) {
        const float* part = a.part + ((long long)(blockIdx.x + k) * 2 + (k ? 0 : 1)) * NR * (HD + 2);
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
      const int R = c0.w + r, j = R / a.group, head = head0 + R - j * a.group;
      const float inv = L == 0.f ? 0.f : V_UP / L;
      T* dst = static_cast<T*>(a.out) + (long long)(c0.y + j) * a.o_ts + (long long)head * a.o_hs + d4 * 4;
      dst[0] = from_f<T>(o.x * inv);
      dst[1] = from_f<T>(o.y * inv);
      dst[2] = from_f<T>(o.z * inv);
      dst[3] = from_f<T>(o.w * inv);
      if (d4 == 0 && a.lse) a.lse[(long long)(c0.y + j) * a.HQ + head] = L == 0.f ? -INFINITY : (mm + log2f(L) - P_EXP<Kind<T>::PS>) * LN2;
    }
    __syncthreads();
  }
}

template <typename T, int HD, int NR, bool PROMPT>
cudaError_t launch_join(const AttnArgs& a, int rows_at_once, cudaStream_t s) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(a.grid, rows_at_once);
  cfg.blockDim = dim3(256);
  cfg.stream = s;
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = at;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, join_kernel<T, HD, NR, PROMPT>, a);
}

}  // namespace

// The prompt kernel (kv4_prompt.cu): 256 rows a tile on the tensor-memory MMAs.
// Its waits give up after `spin` tries.
constexpr int SPIN = 1 << 20;
template <typename T, int HD> cudaError_t launch_prompt(AttnArgs a, int n_sm, int spin, void* ws, cudaStream_t s);
size_t prompt_ws_bytes(int hd, int n_sm);

}  // namespace kv4
}  // namespace bfp
