// kv4.cu -- rotary positions, append and read of the 4-bit paged KV cache
// (record layout and number format in kv4.cuh).
//
// The rotation of a pair (a, b) at position p with frequency f_j is
//   (a c - b s, a s + b c),  c = cos(p f_j), s = sin(p f_j)
// taken from a 32-bit table that the caller builds in 64 bits
// (long-context scalings change only the table).  Products and sums are
// single IEEE operations in 32 bits, rounded once to the output type; the
// inverse (the gradient) negates s.  rope and read are bound by memory; append
// of prompts is not (figures at each kernel).
#include "kv4.cuh"

#include <cstring>
#include <exception>
#include <mutex>
#include <string>
#include <type_traits>

int bfp200_set_error(int code, const std::string& msg);   // engine.cu

namespace bfp {
namespace kv4 {

int device_ready(const char* who, int* n_sm) {
  static std::mutex mu;
  static int sms[128];                        // 0: not asked yet
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return bfp200_set_error(BFP200_ENODEV, std::string(who) + ": " + cudaGetErrorString(e));
  if (dev < 0 || dev >= 128) return bfp200_set_error(BFP200_ENODEV, std::string(who) + ": device index out of range");
  std::lock_guard<std::mutex> lk(mu);
  if (!sms[dev]) {
    int major = 0, n = 0;
    e = cudaDeviceGetAttribute(&major, cudaDevAttrComputeCapabilityMajor, dev);
    if (e == cudaSuccess) e = cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev);
    if (e != cudaSuccess) return bfp200_set_error(BFP200_ECUDA, std::string(who) + ": " + cudaGetErrorString(e));
    if (major != 10) return bfp200_set_error(BFP200_ENODEV, std::string(who) + ": needs an sm_100 (B200) device");
    sms[dev] = n;
  }
  *n_sm = sms[dev];
  return BFP200_OK;
}

int fill_batch(const bfp200_kv4_batch& in, Batch* out, const char* who) {
  const auto bad = [&](const char* what) { return bfp200_set_error(BFP200_EINVAL, std::string(who) + ": " + what); };
  if (in.n_tokens < 0 || in.n_seq < 0 || in.n_pages < 0 || in.max_pages < 0) return bad("negative size");
  if (in.HD != 32 && in.HD != 64 && in.HD != 96 && in.HD != 128) return bad("HD must be 32, 64, 96 or 128");
  if (in.page != 16 && in.page != 32 && in.page != 64 && in.page != 128 && in.page != 256)
    return bad("page must be 16, 32, 64, 128 or 256");
  if (in.H_KV < 1 || in.H_KV > 1024) return bad("H_KV must be 1..1024");
  if (in.n_tokens > (1LL << 30) || in.n_seq > (1LL << 24) || in.n_pages > (1LL << 30))
    return bad("too many tokens, sequences or pages");
  if (in.max_pages > (1LL << 30) / in.page) return bad("a sequence may hold at most 2^30 positions");
  if (in.n_tokens > 0 && in.n_seq > 0 && (!in.q_start_dev || !in.lens_dev)) return bad("q_start and lens are needed");
  if (in.n_tokens > 0 && in.n_seq > 0 && in.max_pages > 0 && !in.block_table_dev) return bad("the block table is needed");
  if (in.n_pages > 0 && !in.pool_dev) return bad("the pool is needed");
  if (reinterpret_cast<uintptr_t>(in.pool_dev) & 15u) return bad("the pool must be 16-byte aligned");
  if ((reinterpret_cast<uintptr_t>(in.q_start_dev) | reinterpret_cast<uintptr_t>(in.lens_dev) |
       reinterpret_cast<uintptr_t>(in.block_table_dev)) & 3u)
    return bad("q_start, lens and the block table must be 4-byte aligned");
  out->pool = static_cast<uint8_t*>(in.pool_dev);
  out->bt = in.block_table_dev;
  out->q_start = in.q_start_dev;
  out->lens = in.lens_dev;
  out->n_pages = (int)in.n_pages;
  out->page = (int)in.page;
  out->page_shift = __builtin_ctzll((unsigned long long)in.page);
  out->H = (int)in.H_KV;
  out->n_seq = (int)in.n_seq;
  out->max_pages = (int)in.max_pages;
  out->T = (int)in.n_tokens;
  out->bt_ld = in.table_stride;
  return BFP200_OK;
}

namespace {

int cuda_fail(const char* who, cudaError_t e) {
  return bfp200_set_error(BFP200_ECUDA, std::string(who) + ": " + cudaGetErrorString(e));
}

__device__ __forceinline__ unsigned u_of(__half2 h) { return *reinterpret_cast<unsigned*>(&h); }
__device__ __forceinline__ unsigned u_of(__nv_bfloat162 h) { return *reinterpret_cast<unsigned*>(&h); }
__device__ __forceinline__ __half2 h2_of(unsigned u) { return *reinterpret_cast<__half2*>(&u); }
__device__ __forceinline__ __nv_bfloat162 b2_of(unsigned u) { return *reinterpret_cast<__nv_bfloat162*>(&u); }

struct Rot {
  const float* table;     // [n_pos][rot / 2][2] (cos, sin)
  const int* positions;   // [T], or null: the token's cache position
  int n_pos, rot;
  bool inter;
};

// (a, b) -> (a c - b s, a s + b c), each product and sum rounded on its own.
__device__ __forceinline__ void turn(float& a, float& b, float c, float s) {
  const float x = __fsub_rn(__fmul_rn(a, c), __fmul_rn(b, s));
  b = __fadd_rn(__fmul_rn(a, s), __fmul_rn(b, c));
  a = x;
}

// ---------------------------------------------------------------------------
// rope: x [T][H][HD] -> out.  One thread keeps the table entries of its dims
// in registers and walks over heads: `VE` dims of a head at a time (both
// halves of the pairs in the half layout).  The unaligned form (VE 1 pair)
// serves any stride.  Bound by memory: 16383 tokens of 40 heads of 128 floats,
// half of the dims turned, 675 MB in 122 us (5.5 TB/s, 84% of the measured copy).
// ---------------------------------------------------------------------------
struct RopeArgs {
  const void* x;
  void* out;
  const float* table;
  const int* pos;
  long long x_ts, x_hs, o_ts, o_hs;
  int T, H, HD, rot, n_pos, tasks, hsplit;   // tasks per head; head groups per token
  float sign;
};

template <typename T, int VE, bool INTER, bool ALIGNED, bool NC>
__global__ void __launch_bounds__(256) rope_kernel(const RopeArgs a) {
  const long long id = (long long)blockIdx.x * blockDim.x + threadIdx.x;
  const int per = a.tasks * a.hsplit;
  const long long t = id / per;
  if (t >= a.T) return;
  const int r = (int)(id - t * per), task = r % a.tasks, hg = r / a.tasks;
  const int per_h = (a.H + a.hsplit - 1) / a.hsplit;
  const int h0 = hg * per_h, h1 = min(a.H, h0 + per_h);
  const T* x = static_cast<const T*>(a.x) + t * a.x_ts;
  T* o = static_cast<T*>(a.out) + t * a.o_ts;
  const int p = min(max(__ldg(a.pos + t), 0), a.n_pos - 1);
  const float* row = a.table + (long long)p * a.rot;
  constexpr int NP = INTER ? (VE > 1 ? VE / 2 : 1) : VE;      // pairs of one thread
  constexpr int W = INTER && VE == 1 ? 2 : VE;                // elements of one vector
  const int rot_tasks = a.rot / (INTER ? W : 2 * W);
  if (task < rot_tasks) {
    float c[NP], s[NP];
    #pragma unroll
    for (int i = 0; i < NP; ++i) {
      const float2 cs = __ldg(reinterpret_cast<const float2*>(row) + task * NP + i);
      c[i] = cs.x;
      s[i] = cs.y * a.sign;
    }
    const int d = task * W;
    #pragma unroll 4
    for (int h = h0; h < h1; ++h) {
      if constexpr (INTER) {
        float v[W];
        load_vec<T, W, ALIGNED, NC>(x + h * a.x_hs + d, v);
        #pragma unroll
        for (int i = 0; i < NP; ++i) turn(v[2 * i], v[2 * i + 1], c[i], s[i]);
        store_vec<T, W, ALIGNED>(o + h * a.o_hs + d, v);
      } else {
        float v[W], w[W];
        load_vec<T, W, ALIGNED, NC>(x + h * a.x_hs + d, v);
        load_vec<T, W, ALIGNED, NC>(x + h * a.x_hs + d + a.rot / 2, w);
        #pragma unroll
        for (int i = 0; i < NP; ++i) turn(v[i], w[i], c[i], s[i]);
        store_vec<T, W, ALIGNED>(o + h * a.o_hs + d, v);
        store_vec<T, W, ALIGNED>(o + h * a.o_hs + d + a.rot / 2, w);
      }
    }
  } else {
    const int d = a.rot + (task - rot_tasks) * W;             // dims that are not rotated
    #pragma unroll 4
    for (int h = h0; h < h1; ++h) {
      if constexpr (ALIGNED) {
        float v[W];
        load_vec<T, W, true, NC>(x + h * a.x_hs + d, v);
        store_vec<T, W, true>(o + h * a.o_hs + d, v);
      } else {
        #pragma unroll
        for (int i = 0; i < W; ++i)
          if (d + i < a.HD) o[h * a.o_hs + d + i] = x[h * a.x_hs + d + i];
      }
    }
  }
}

template <typename T>
cudaError_t launch_rope(RopeArgs a, bool inter, cudaStream_t s) {
  constexpr int VE = 16 / (int)sizeof(T);
  const auto al = [](long long v) { return v % VE == 0; };
  const bool aligned = al(a.x_ts) && al(a.x_hs) && al(a.o_ts) && al(a.o_hs) && a.HD % VE == 0 &&
                       a.rot % (inter ? VE : 2 * VE) == 0 && reinterpret_cast<uintptr_t>(a.x) % 16 == 0 &&
                       reinterpret_cast<uintptr_t>(a.out) % 16 == 0;
  const int w = aligned ? VE : inter ? 2 : 1;
  a.tasks = a.rot / (inter ? w : 2 * w) + (a.HD - a.rot + w - 1) / w;
  // Table entries are reused across the heads of a thread; heads are split
  // over threads only while the GPU is not full.
  a.hsplit = 1;
  while (a.hsplit < a.H && (long long)a.T * a.tasks * a.hsplit < 148LL * 2048) a.hsplit *= 2;
  a.hsplit = a.hsplit < a.H ? a.hsplit : a.H;
  const long long threads = (long long)a.T * a.tasks * a.hsplit, blocks = (threads + 255) / 256;
  if (blocks > 0x7fffffffLL) return cudaErrorInvalidConfiguration;
  const dim3 g((unsigned)blocks);
  const bool apart = a.x != a.out;              // not in place: the read-only path (16383 x 40 x 128 floats: 122 us, else 133)
  if (aligned && inter) (apart ? rope_kernel<T, VE, true, true, true> : rope_kernel<T, VE, true, true, false>)<<<g, 256, 0, s>>>(a);
  else if (aligned) (apart ? rope_kernel<T, VE, false, true, true> : rope_kernel<T, VE, false, true, false>)<<<g, 256, 0, s>>>(a);
  else if (inter) rope_kernel<T, 1, true, false, false><<<g, 256, 0, s>>>(a);
  else rope_kernel<T, 1, false, false, false><<<g, 256, 0, s>>>(a);
  return cudaGetLastError();
}

// ---------------------------------------------------------------------------
// append: a warp takes rows of one token (keys, values, then queries), LPR
// lanes a row, 8 dims a lane; two lanes hold a tile.  The token's table entries
// stay in registers over the rows, and the rows' loads are issued before the
// token's place is looked up.  A row's nibbles go straight to their record: the
// 4-byte (keys) and 2-byte (values) pieces of neighbouring tokens meet in L2.
// 26.8k tokens of 32 / 8 heads of 128 float16: 152 us, 531 MB of DRAM traffic
// (3.5 TB/s), 60% of the issue slots at 35% of the warps, of whose stalls the
// loads' latency is the largest part: neither instructions nor memory are at a
// limit by themselves.  Appending and reading back take 180 us so, 217
// before a pass held rows of one kind only, 207 at 2 CTAs an SM instead of 3 (more
// registers a thread), 184 at 4 with half the rows in flight.
// ---------------------------------------------------------------------------
struct AppendArgs {
  Batch b;
  Rot r;
  const void *k, *v, *q;
  void* q_out;
  long long k_ts, k_hs, v_ts, v_hs, q_ts, q_hs, o_ts, o_hs;
  int HQ, passes, groups, group_passes;     // groups of passes of a token, one a warp
  int table_vec;                            // table rows can be read 16 bytes at a time
};

template <int HD> constexpr int LANES_PER_ROW = HD <= 32 ? 4 : HD <= 64 ? 8 : 16;

// 8 elements as they lie in memory.
template <typename T> struct Raw8 { unsigned w[2 * sizeof(T)]; };
template <typename T, bool ALIGNED>
__device__ __forceinline__ Raw8<T> load_raw(const T* p) {
  Raw8<T> r;
  if constexpr (ALIGNED) {
    #pragma unroll
    for (int i = 0; i < (int)sizeof(T) / 2; ++i) {
      const uint4 v = __ldcs(reinterpret_cast<const uint4*>(p) + i);
      r.w[4 * i] = v.x; r.w[4 * i + 1] = v.y; r.w[4 * i + 2] = v.z; r.w[4 * i + 3] = v.w;
    }
  } else if constexpr (sizeof(T) == 4) {
    #pragma unroll
    for (int i = 0; i < 8; ++i) r.w[i] = __ldcs(reinterpret_cast<const unsigned*>(p) + i);
  } else {
    const unsigned short* h = reinterpret_cast<const unsigned short*>(p);
    #pragma unroll
    for (int i = 0; i < 4; ++i) r.w[i] = __ldcs(h + 2 * i) | (unsigned)__ldcs(h + 2 * i + 1) << 16;
  }
  return r;
}
template <typename T>
__device__ __forceinline__ void to_floats(const Raw8<T>& r, float (&f)[8]) {
  if constexpr (sizeof(T) == 4) {
    #pragma unroll
    for (int i = 0; i < 8; ++i) f[i] = __uint_as_float(r.w[i]);
  } else {
    #pragma unroll
    for (int i = 0; i < 4; ++i) {
      T e[2];
      memcpy(e, &r.w[i], 4);
      f[2 * i] = to_f(e[0]);
      f[2 * i + 1] = to_f(e[1]);
    }
  }
}

// The sequence of token t (see find_seq); in a step of one token each it is t.
__device__ __forceinline__ int seq_of_token(const Batch& b, int t) {
  if (b.T == b.n_seq && __ldg(b.q_start + t) == t && __ldg(b.q_start + t + 1) == t + 1) return t;
  return find_seq(b.q_start, b.n_seq, t);
}

template <typename T, int HD, bool ALIGNED>
__global__ void __launch_bounds__(256, sizeof(T) == 4 ? 2 : 3) append_kernel(const AppendArgs a) {
  constexpr int LPR = LANES_PER_ROW<HD>, RPW = 32 / LPR, REC9 = HD * 9 / 8, UNR = 4;
  __shared__ float s_exch[8][RPW][HD];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int li = lane % LPR, ri = lane / LPR, d0 = li * 8;
  const long long wid = (long long)blockIdx.x * 8 + warp;
  const int t = (int)(wid / a.groups), grp = (int)(wid - (long long)t * a.groups);
  if (t >= a.b.T) return;
  // A pass is RPW rows of one kind: PH passes of keys, PH of values, then queries.
  const int H = a.b.H, PH = (H + RPW - 1) / RPW, p_end = min(a.passes, (grp + 1) * a.group_passes);
  const T* const kb = static_cast<const T*>(a.k) + t * a.k_ts + d0;
  const T* const vb = static_cast<const T*>(a.v) + t * a.v_ts + d0;
  const T* const qb = static_cast<const T*>(a.q) + t * a.q_ts + d0;
  T* const ob = static_cast<T*>(a.q_out) + t * a.o_ts + d0;
  Raw8<T> raw[UNR];
  const auto load = [&](int p0) {
    #pragma unroll
    for (int k = 0; k < UNR; ++k) {
      const int p = p0 + k;
      if (p >= p_end) break;
      const int h = (p < PH ? p : p < 2 * PH ? p - PH : p - 2 * PH) * RPW + ri;
      raw[k] = Raw8<T>{};
      if (d0 < HD && h < (p < 2 * PH ? H : a.HQ))
        raw[k] = load_raw<T, ALIGNED>(p < PH ? kb + h * a.k_hs : p < 2 * PH ? vb + h * a.v_hs : qb + h * a.q_hs);
    }
  };
  load(grp * a.group_passes);
  int seq = 0, q_end = 0, pos = -1;
  bool held = false;
  if (a.b.n_seq) {
    seq = seq_of_token(a.b, t);
    q_end = __ldg(a.b.q_start + seq + 1);
    pos = __ldg(a.b.lens + seq) - q_end + t;
    held = t >= __ldg(a.b.q_start + seq) && t < q_end && pos >= 0 && (pos >> a.b.page_shift) < a.b.max_pages;
  }
  const int pg = held ? __ldg(a.b.bt + (long long)seq * a.b.bt_ld + (pos >> a.b.page_shift)) : -1;
  const bool store = held && (unsigned)pg < (unsigned)a.b.n_pages;
  const int rot = a.r.table ? a.r.rot : 0, half = rot >> 1;
  // The lane's (cos, sin): of its 4 pairs (interleaved), or one for each of its
  // dims, the sign of sin turned where the dim is the first of its pair.
  const bool lanewise = (half & 7) == 0;                    // the pair's other dims are a whole lane's
  float c[8], sn[8];
  if (rot) {
    const int p = a.r.positions ? __ldg(a.r.positions + t) : pos;
    const float* row = a.r.table + (long long)min(max(p, 0), a.r.n_pos - 1) * rot;
    if (a.r.inter) {
      #pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float2 cs = d0 + 2 * i < rot ? __ldg(reinterpret_cast<const float2*>(row) + d0 / 2 + i) : make_float2(1.f, 0.f);
        c[i] = cs.x;
        sn[i] = cs.y;
      }
    } else if (lanewise && a.table_vec && d0 < rot) {
      const float4* cs4 = reinterpret_cast<const float4*>(row + (d0 < half ? d0 : d0 - half) * 2);
      const float sign = d0 < half ? -1.f : 1.f;
      #pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float4 v = __ldg(cs4 + i);
        c[2 * i] = v.x; c[2 * i + 1] = v.z;
        sn[2 * i] = v.y * sign; sn[2 * i + 1] = v.w * sign;
      }
    } else {
      #pragma unroll
      for (int i = 0; i < 8; ++i) {
        const int d = d0 + i;
        const float2 cs = d < rot ? __ldg(reinterpret_cast<const float2*>(row) + (d < half ? d : d - half)) : make_float2(1.f, 0.f);
        c[i] = cs.x;
        sn[i] = d < half ? -cs.y : cs.y;
      }
    }
  }
  const int src = !lanewise || d0 >= rot ? lane : d0 < half ? lane + (half >> 3) : lane - (half >> 3);
  // a row turned, as floats
  const auto rotate = [&](const Raw8<T>& r, float (&f)[8]) {
    to_floats(r, f);
    if (!rot) return;
    if (a.r.inter) {
      #pragma unroll
      for (int i = 0; i < 4; ++i)
        if (d0 + 2 * i < rot) turn(f[2 * i], f[2 * i + 1], c[i], sn[i]);
    } else if (lanewise) {
      Raw8<T> other;
      #pragma unroll
      for (int i = 0; i < (int)(2 * sizeof(T)); ++i) other.w[i] = __shfl_sync(0xffffffffu, r.w[i], src);
      float o[8];                                           // the other elements of the pairs
      to_floats(other, o);
      if (d0 < rot) {
        #pragma unroll
        for (int i = 0; i < 8; ++i) f[i] = __fadd_rn(__fmul_rn(f[i], c[i]), __fmul_rn(o[i], sn[i]));   // a c - b s, or b c + a s
      }
    } else {
      float* exch = s_exch[warp][ri];
      #pragma unroll
      for (int i = 0; i < 8; ++i)
        if (d0 + i < HD) exch[d0 + i] = f[i];
      __syncwarp();
      #pragma unroll
      for (int i = 0; i < 8; ++i) {
        const int d = d0 + i;
        if (d < rot) f[i] = __fadd_rn(__fmul_rn(f[i], c[i]), __fmul_rn(exch[d < half ? d + half : d - half], sn[i]));
      }
      __syncwarp();
    }
  };
  // the row's 8 nibbles of this lane, and their tile's exponent byte
  const auto quantize = [&](const float (&f)[8], int& e) {
    float top = 0.f;
    #pragma unroll
    for (int i = 0; i < 8; ++i) top = fmaxf(top, fabsf(f[i]));
    top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
    e = tile_e(top);
    const float up = pow2f(3 - e);
    unsigned w = 0;                                         // sum of m_i 16^i modulo 2^32; adding 8 to every nibble makes them 0..15
    #pragma unroll
    for (int i = 7; i >= 0; --i) w = w * 16 + (unsigned)mantissa(f[i], up);
    return w + 0x88888888u;
  };
  const int slot = pos & (a.b.page - 1), page = a.b.page;
  uint8_t* const rec0 = a.b.pool + (store ? (long long)pg * H : 0) * (page * REC9);
  uint8_t* const k_at = rec0 + ((slot >> 2) * (HD / 8) + li) * 16 + (slot & 3) * 4;
  uint8_t* const v_at = rec0 + page * HD / 2 + ((slot >> 3) * (HD / 4) + 2 * li) * 16 + (slot & 3) * 4 + (slot >> 2 & 1) * 2;
  uint8_t* const e_at = rec0 + page * HD + li / 2 * page + slot;
  #pragma unroll 1
  for (int p0 = grp * a.group_passes; p0 < p_end; p0 += UNR) {
    if (p0 != grp * a.group_passes) load(p0);
    #pragma unroll
    for (int k = 0; k < UNR; ++k) {
      const int p = p0 + k;
      if (p >= p_end) break;
      float f[8];
      if (p >= 2 * PH) {                                    // queries
        const int h = (p - 2 * PH) * RPW + ri;
        rotate(raw[k], f);
        if (d0 < HD && h < a.HQ) store_vec<T, 8, ALIGNED>(ob + h * a.o_hs, f);
      } else {
        const bool key = p < PH;
        const int h = (key ? p : p - PH) * RPW + ri;
        if (key) rotate(raw[k], f);
        else to_floats(raw[k], f);
        int e;
        const unsigned w = quantize(f, e);
        if (!store || d0 >= HD || h >= H) continue;
        const int off = h * (page * REC9);
        if (key) {
          *reinterpret_cast<unsigned*>(k_at + off) = w;
        } else {
          *reinterpret_cast<uint16_t*>(v_at + off) = (uint16_t)w;
          *reinterpret_cast<uint16_t*>(v_at + off + 16) = (uint16_t)(w >> 16);
        }
        if ((li & 1) == 0) e_at[off + (key ? 0 : HD / 16 * page)] = (uint8_t)(e + 18);
      }
    }
  }
}

// ---------------------------------------------------------------------------
// read: a warp decodes octs of 8 positions, HD / 4 lanes a head: a key unit (4
// positions x 8 dims) and a value unit (8 positions x 4 dims) a lane, 16 bytes
// each.  An oct belongs to the warp that holds its first token.  16 sequences of
// up to 8192 positions, 8 heads of 128, to float16: 355 MB in 64 us (5.5 TB/s,
// 84% of the measured copy; 61% of the ALU).  The first form, which read 4, 2 and
// 1 bytes at a time, took 86 us.
// ---------------------------------------------------------------------------
struct ReadArgs {
  Batch b;
  void *k, *v;          // [T][H][HD]
  int span;             // tokens of a warp
};

// 8 nibbles of a word times the 16-bit scales of its halves (2^(B - 21)), as the
// pairs (n, n + 4); exact in both types.
template <typename T>
__device__ __forceinline__ void nibble_pairs(unsigned w, unsigned bytes, unsigned (&o)[4]) {
  if constexpr (std::is_same<T, __half>::value) {
    // 2^(B - 15) 2^-6 (the mask keeps a byte that stands for no position out of the other half)
    const __half2 h = __hmul2(h2_of(bytes << 10 & 0x7C007C00u), __floats2half2_rn(0x1p-6f, 0x1p-6f));
    #pragma unroll
    for (int n = 0; n < 4; ++n)
      o[n] = u_of(__hmul2(__hsub2(h2_of((w >> (4 * n) & 0x000F000Fu) | 0x64006400u), __floats2half2_rn(1032.f, 1032.f)), h));
  } else {
    const unsigned s = bytes * 128u + 0x35003500u;
    const __nv_bfloat162 sc = b2_of(s), c = __hmul2(sc, __floats2bfloat162_rn(-136.f, -136.f));
    #pragma unroll
    for (int n = 0; n < 4; ++n) o[n] = u_of(__hfma2(b2_of((w >> (4 * n) & 0x000F000Fu) | 0x43004300u), sc, c));
  }
}
// N pairs of 16-bit values to T (bfloat16 pairs widen to float by a shift).
template <typename T, int N>
__device__ __forceinline__ void put(T* p, const unsigned (&v)[N]) {
  if constexpr (std::is_same<T, float>::value) {
    #pragma unroll
    for (int i = 0; i < N; i += 2)
      *reinterpret_cast<uint4*>(p + 2 * i) = make_uint4(v[i] << 16, v[i] & 0xFFFF0000u, v[i + 1] << 16, v[i + 1] & 0xFFFF0000u);
  } else if constexpr (N == 4) {
    *reinterpret_cast<uint4*>(p) = make_uint4(v[0], v[1], v[2], v[3]);
  } else {
    *reinterpret_cast<uint2*>(p) = make_uint2(v[0], v[1]);
  }
}

template <typename T, int HD>
__global__ void __launch_bounds__(256) read_kernel(const ReadArgs a) {
  constexpr int REC9 = HD * 9 / 8, LH = HD / 4, HPW = 32 / LH;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int H = a.b.H, page = a.b.page, hg = (H + HPW - 1) / HPW;
  const long long wid = (long long)blockIdx.x * 8 + warp;
  const long long t0 = wid / hg * a.span;
  const int sub = lane / LH, u = lane % LH, h = (int)(wid % hg) * HPW + sub;
  if (t0 >= a.b.T) return;
  const int t_end = (int)min((long long)a.b.T, t0 + a.span);
  const bool on = sub < HPW && h < H;
  int seq = find_seq(a.b.q_start, a.b.n_seq, (int)t0);
  int t = (int)t0;
  while (t < t_end) {                                       // the same for every lane
    while (seq + 1 < a.b.n_seq && __ldg(a.b.q_start + seq + 1) <= t) ++seq;
    const int q0 = __ldg(a.b.q_start + seq), q1 = __ldg(a.b.q_start + seq + 1);
    const int pos = __ldg(a.b.lens + seq) - q1 + t;
    const bool mine = t >= q0 && t < q1 && pos >= 0 && (pos >> a.b.page_shift) < a.b.max_pages;
    if (!mine) {                                            // a token without a place reads as zeros
      const unsigned z[4] = {0, 0, 0, 0};
      if (on && u < HD / 8) {
        put<T, 4>(static_cast<T*>(a.k) + ((long long)t * H + h) * HD + u * 8, z);
        put<T, 4>(static_cast<T*>(a.v) + ((long long)t * H + h) * HD + u * 8, z);
      }
      ++t;
      continue;
    }
    if (t > q0 && (pos & 7)) { ++t; continue; }             // inside an oct of another warp's, or of the last round
    const int o = pos & 7, n = min(min(8 - o, q1 - t), a.b.T - t);   // tokens t .. t + n - 1 at places o .. o + n - 1 of the oct
    const int pg = __ldg(a.b.bt + (long long)seq * a.b.bt_ld + (pos >> a.b.page_shift));
    const bool there = (unsigned)pg < (unsigned)a.b.n_pages;
    const int slot = pos & (page - 8);
    if (on) {
      const uint8_t* rec = a.b.pool + (there ? ((long long)pg * H + h) * (page * REC9) : 0);
      uint4 kw, vw;
      unsigned ke;
      uint2 ve;
      const int quad = u / (HD / 8), ku = u % (HD / 8);
      if (there) {
        kw = __ldg(reinterpret_cast<const uint4*>(rec + ((slot >> 2) * (HD / 8) + u) * 16));
        vw = __ldg(reinterpret_cast<const uint4*>(rec + page * HD / 2 + ((slot >> 3) * (HD / 4) + u) * 16));
        ke = __ldg(reinterpret_cast<const unsigned*>(rec + page * HD + (ku >> 1) * page + slot + 4 * quad));
        ve = __ldg(reinterpret_cast<const uint2*>(rec + page * HD + (HD / 16 + (u >> 2)) * page + slot));
      } else {
        kw = vw = make_uint4(0x88888888u, 0x88888888u, 0x88888888u, 0x88888888u);
        ke = 0x15151515u;
        ve = make_uint2(0x15151515u, 0x15151515u);
      }
      const unsigned kword[4] = {kw.x, kw.y, kw.z, kw.w}, vword[4] = {vw.x, vw.y, vw.z, vw.w};
      T* kp = static_cast<T*>(a.k) + ((long long)(t - o) * H + h) * HD + ku * 8;
      T* vp = static_cast<T*>(a.v) + ((long long)(t - o) * H + h) * HD + u * 4;
      #pragma unroll
      for (int i = 0; i < 4; ++i) {
        unsigned op[4];
        const unsigned kb = (ke >> (8 * i) & 0xFFu) * 0x10001u;
        nibble_pairs<T>(kword[i], kb, op);
        const unsigned row[4] = {__byte_perm(op[0], op[1], 0x5410), __byte_perm(op[2], op[3], 0x5410),
                                 __byte_perm(op[0], op[1], 0x7632), __byte_perm(op[2], op[3], 0x7632)};
        const int pk = 4 * quad + i;
        if (pk >= o && pk < o + n) put<T, 4>(kp + (long long)pk * H * HD, row);
        nibble_pairs<T>(vword[i], (ve.x >> (8 * i) & 0xFFu) | (ve.y >> (8 * i) & 0xFFu) << 16, op);
        const unsigned lo[2] = {__byte_perm(op[0], op[1], 0x5410), __byte_perm(op[2], op[3], 0x5410)};
        const unsigned hi[2] = {__byte_perm(op[0], op[1], 0x7632), __byte_perm(op[2], op[3], 0x7632)};
        if (i >= o && i < o + n) put<T, 2>(vp + (long long)i * H * HD, lo);
        if (i + 4 >= o && i + 4 < o + n) put<T, 2>(vp + (long long)(i + 4) * H * HD, hi);
      }
    }
    t += n;
  }
}

template <typename T, int HD>
cudaError_t launch_append(AppendArgs a, bool aligned, cudaStream_t s) {
  constexpr int RPW = 32 / LANES_PER_ROW<HD>;
  a.passes = 2 * ((a.b.H + RPW - 1) / RPW) + (a.HQ + RPW - 1) / RPW;
  // All rows of a token by one warp, or batches of 4 passes by several while the GPU has room.
  int batches = (a.passes + 3) / 4, each = batches;
  while (each > 1 && (long long)a.b.T * ((batches + each - 1) / each) < 148LL * 32) each = (each + 1) / 2;
  a.group_passes = each * 4;
  a.groups = (batches + each - 1) / each;
  a.table_vec = a.r.table && a.r.rot % 4 == 0 && reinterpret_cast<uintptr_t>(a.r.table) % 16 == 0;
  const long long blocks = ((long long)a.b.T * a.groups + 7) / 8;
  if (blocks > 0x7fffffffLL) return cudaErrorInvalidConfiguration;
  if (aligned) append_kernel<T, HD, true><<<(unsigned)blocks, 256, 0, s>>>(a);
  else append_kernel<T, HD, false><<<(unsigned)blocks, 256, 0, s>>>(a);
  return cudaGetLastError();
}

template <typename T, int HD>
cudaError_t launch_read(ReadArgs a, cudaStream_t s) {
  constexpr int HPW = 32 / (HD / 4);
  const long long hg = (a.b.H + HPW - 1) / HPW;
  // 8 tokens a warp are one oct of a prompt, but 8 octs of a step's sequences:
  // one after the other only where the GPU is full without.
  a.span = a.b.T * hg <= 148LL * 64 ? 1 : 8;
  const long long blocks = (((long long)a.b.T + a.span - 1) / a.span * hg + 7) / 8;
  if (blocks > 0x7fffffffLL) return cudaErrorInvalidConfiguration;
  read_kernel<T, HD><<<(unsigned)blocks, 256, 0, s>>>(a);
  return cudaGetLastError();
}

template <typename F> cudaError_t by_hd(int hd, F f) {
  switch (hd) {
    case 32: return f(std::integral_constant<int, 32>{});
    case 64: return f(std::integral_constant<int, 64>{});
    case 96: return f(std::integral_constant<int, 96>{});
    default: return f(std::integral_constant<int, 128>{});
  }
}

int elem_size(long long dtype) { return dtype == BFP200_F32 ? 4 : dtype == BFP200_F16 || dtype == BFP200_BF16 ? 2 : 0; }

}  // namespace
}  // namespace kv4
}  // namespace bfp

using namespace bfp::kv4;

extern "C" int bfp200_rope_dev(const bfp200_rope_args* in, void* stream) try {
  const char* who = "rope_dev";
  const auto bad = [&](const char* what) { return bfp200_set_error(BFP200_EINVAL, std::string(who) + ": " + what); };
  if (!in) return bad("no arguments");
  const bfp200_rope_args& r = *in;
  if (!elem_size(r.dtype)) return bad("dtype must be BFP200_F32, BFP200_F16 or BFP200_BF16");
  if (r.T < 0 || r.H < 0 || r.T > (1LL << 30) || r.H > (1LL << 20)) return bad("bad number of tokens or heads");
  if (r.HD < 1 || r.HD > 4096) return bad("HD must be 1..4096");
  if (r.rot < 0 || r.rot > r.HD || r.rot % 2) return bad("rot must be even and at most HD");
  if (r.n_pos < 1 || r.n_pos > (1LL << 30)) return bad("the table needs at least one position");
  if (!r.T || !r.H) return BFP200_OK;
  if (!r.x_dev || !r.out_dev || !r.positions_dev || (r.rot && !r.table_dev)) return bad("null pointer");
  if (reinterpret_cast<uintptr_t>(r.table_dev) & 7u) return bad("the table must be 8-byte aligned");
  if (reinterpret_cast<uintptr_t>(r.positions_dev) & 3u) return bad("positions must be 4-byte aligned");
  const int es = elem_size(r.dtype);
  if ((reinterpret_cast<uintptr_t>(r.x_dev) | reinterpret_cast<uintptr_t>(r.out_dev)) % es) return bad("misaligned x or out");
  int n_sm = 0;
  if (int rc = device_ready(who, &n_sm)) return rc;
  RopeArgs a;
  a.x = r.x_dev; a.out = r.out_dev; a.table = r.table_dev; a.pos = r.positions_dev;
  a.x_ts = r.x_ts; a.x_hs = r.x_hs; a.o_ts = r.o_ts; a.o_hs = r.o_hs;
  a.T = (int)r.T; a.H = (int)r.H; a.HD = (int)r.HD; a.rot = (int)r.rot; a.n_pos = (int)r.n_pos;
  a.sign = r.inverse ? -1.f : 1.f;
  a.tasks = a.hsplit = 0;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const cudaError_t e = r.dtype == BFP200_F32 ? launch_rope<float>(a, r.interleaved != 0, s)
                      : r.dtype == BFP200_F16 ? launch_rope<__half>(a, r.interleaved != 0, s)
                                              : launch_rope<__nv_bfloat16>(a, r.interleaved != 0, s);
  return e == cudaSuccess ? BFP200_OK : cuda_fail(who, e);
} catch (const std::exception& ex) {
  return bfp200_set_error(BFP200_ENOMEM, ex.what());
}

extern "C" int bfp200_kv4_append_dev(const bfp200_kv4_append_args* in, void* stream) try {
  const char* who = "kv4_append_dev";
  const auto bad = [&](const char* what) { return bfp200_set_error(BFP200_EINVAL, std::string(who) + ": " + what); };
  if (!in) return bad("no arguments");
  const bfp200_kv4_append_args& r = *in;
  AppendArgs a;
  if (int rc = fill_batch(r.batch, &a.b, who)) return rc;
  const int es = elem_size(r.dtype), HD = (int)r.batch.HD;
  if (!es) return bad("dtype must be BFP200_F32, BFP200_F16 or BFP200_BF16");
  if (r.H_Q < 0 || r.H_Q > (1LL << 16)) return bad("bad number of query heads");
  if (r.table_dev) {
    if (r.rot < 0 || r.rot > HD || r.rot % 2) return bad("rot must be even and at most HD");
    if (r.n_pos < 1 || r.n_pos > (1LL << 30)) return bad("the table needs at least one position");
    if (!r.positions_dev && r.n_pos < r.batch.max_pages * r.batch.page)
      return bad("the rotation table is shorter than max_pages * page positions");
    if (reinterpret_cast<uintptr_t>(r.table_dev) & 7u) return bad("the table must be 8-byte aligned");
    if (reinterpret_cast<uintptr_t>(r.positions_dev) & 3u) return bad("positions must be 4-byte aligned");
  }
  if (a.b.T == 0 || (a.b.n_seq == 0 && r.H_Q == 0)) return BFP200_OK;
  if (!r.k_dev || !r.v_dev || (r.H_Q > 0 && (!r.q_dev || !r.q_out_dev))) return bad("null pointer");
  const uintptr_t all = reinterpret_cast<uintptr_t>(r.k_dev) | reinterpret_cast<uintptr_t>(r.v_dev) |
                        (r.H_Q ? reinterpret_cast<uintptr_t>(r.q_dev) | reinterpret_cast<uintptr_t>(r.q_out_dev) : 0);
  if (all % es) return bad("misaligned k, v or q");
  int n_sm = 0;
  if (int rc = device_ready(who, &n_sm)) return rc;
  a.r.table = r.table_dev; a.r.positions = r.positions_dev; a.r.n_pos = (int)r.n_pos; a.r.rot = (int)r.rot;
  a.r.inter = r.interleaved != 0;
  a.k = r.k_dev; a.v = r.v_dev; a.q = r.q_dev; a.q_out = r.q_out_dev;
  a.k_ts = r.k_ts; a.k_hs = r.k_hs; a.v_ts = r.v_ts; a.v_hs = r.v_hs;
  a.q_ts = r.q_ts; a.q_hs = r.q_hs; a.o_ts = r.o_ts; a.o_hs = r.o_hs;
  a.HQ = (int)r.H_Q;
  a.passes = a.groups = a.group_passes = a.table_vec = 0;
  long long strides = r.k_ts | r.k_hs | r.v_ts | r.v_hs;
  if (r.H_Q) strides |= r.q_ts | r.q_hs | r.o_ts | r.o_hs;
  const bool aligned = all % 16 == 0 && strides * es % 16 == 0;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const cudaError_t e = by_hd(HD, [&](auto hd) {
    constexpr int N = decltype(hd)::value;
    return r.dtype == BFP200_F32 ? launch_append<float, N>(a, aligned, s)
         : r.dtype == BFP200_F16 ? launch_append<__half, N>(a, aligned, s)
                                 : launch_append<__nv_bfloat16, N>(a, aligned, s);
  });
  return e == cudaSuccess ? BFP200_OK : cuda_fail(who, e);
} catch (const std::exception& ex) {
  return bfp200_set_error(BFP200_ENOMEM, ex.what());
}

extern "C" int bfp200_kv4_read_dev(const bfp200_kv4_read_args* in, void* stream) try {
  const char* who = "kv4_read_dev";
  const auto bad = [&](const char* what) { return bfp200_set_error(BFP200_EINVAL, std::string(who) + ": " + what); };
  if (!in) return bad("no arguments");
  ReadArgs a;
  if (int rc = fill_batch(in->batch, &a.b, who)) return rc;
  if (!elem_size(in->dtype)) return bad("dtype must be BFP200_F32, BFP200_F16 or BFP200_BF16");
  if (a.b.T == 0) return BFP200_OK;
  if (!in->k_out_dev || !in->v_out_dev) return bad("null pointer");
  if ((reinterpret_cast<uintptr_t>(in->k_out_dev) | reinterpret_cast<uintptr_t>(in->v_out_dev)) & 15u)
    return bad("outputs must be 16-byte aligned");
  int n_sm = 0;
  if (int rc = device_ready(who, &n_sm)) return rc;
  a.k = in->k_out_dev; a.v = in->v_out_dev;
  a.span = 0;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (a.b.n_seq == 0) {                                     // tokens of no sequence
    const size_t bytes = (size_t)a.b.T * a.b.H * (size_t)in->batch.HD * elem_size(in->dtype);
    cudaError_t z = cudaMemsetAsync(a.k, 0, bytes, s);
    if (z == cudaSuccess) z = cudaMemsetAsync(a.v, 0, bytes, s);
    return z == cudaSuccess ? BFP200_OK : cuda_fail(who, z);
  }
  const cudaError_t e = by_hd((int)in->batch.HD, [&](auto hd) {
    constexpr int N = decltype(hd)::value;
    return in->dtype == BFP200_F32 ? launch_read<float, N>(a, s)
         : in->dtype == BFP200_F16 ? launch_read<__half, N>(a, s)
                                   : launch_read<__nv_bfloat16, N>(a, s);
  });
  return e == cudaSuccess ? BFP200_OK : cuda_fail(who, e);
} catch (const std::exception& ex) {
  return bfp200_set_error(BFP200_ENOMEM, ex.what());
}
