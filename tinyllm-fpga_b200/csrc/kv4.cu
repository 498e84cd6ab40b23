// kv4.cu -- rotary positions, append and read of the 4-bit paged KV cache
// (record layout and number format in kv4.cuh).
//
// The rotation of a pair (a, b) at position p with frequency f_j is
//   (a c - b s, a s + b c),  c = cos(p f_j), s = sin(p f_j)
// taken from a 32-bit table that the caller builds in 64 bits
// (long-context scalings change only the table).  Products and sums are
// single IEEE operations in 32 bits, rounded once to the output type; the
// inverse (the gradient) negates s.  All three kernels are bound by memory.
#include "kv4.cuh"

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
  if (in.max_pages * in.page > (1LL << 30)) return bad("a sequence may hold at most 2^30 positions");
  if (in.n_tokens > 0 && in.n_seq > 0 && (!in.q_start_dev || !in.lens_dev)) return bad("q_start and lens are needed");
  if (in.n_tokens > 0 && in.n_seq > 0 && in.max_pages > 0 && !in.block_table_dev) return bad("the block table is needed");
  if (in.n_pages > 0 && !in.pool_dev) return bad("the pool is needed");
  if (reinterpret_cast<uintptr_t>(in.pool_dev) & 15u) return bad("the pool must be 16-byte aligned");
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
// serves any stride.
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

template <typename T, int VE, bool INTER, bool ALIGNED>
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
        load_vec<T, W, ALIGNED>(x + h * a.x_hs + d, v);
        #pragma unroll
        for (int i = 0; i < NP; ++i) turn(v[2 * i], v[2 * i + 1], c[i], s[i]);
        store_vec<T, W, ALIGNED>(o + h * a.o_hs + d, v);
      } else {
        float v[W], w[W];
        load_vec<T, W, ALIGNED>(x + h * a.x_hs + d, v);
        load_vec<T, W, ALIGNED>(x + h * a.x_hs + d + a.rot / 2, w);
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
        load_vec<T, W, true>(x + h * a.x_hs + d, v);
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
  if (aligned && inter) rope_kernel<T, VE, true, true><<<g, 256, 0, s>>>(a);
  else if (aligned) rope_kernel<T, VE, false, true><<<g, 256, 0, s>>>(a);
  else if (inter) rope_kernel<T, 1, true, false><<<g, 256, 0, s>>>(a);
  else rope_kernel<T, 1, false, false><<<g, 256, 0, s>>>(a);
  return cudaGetLastError();
}

// ---------------------------------------------------------------------------
// append: rows of a token (keys, values, then queries) are taken by groups of
// LPR lanes, 8 dims a lane; two lanes hold a tile.
// ---------------------------------------------------------------------------
struct AppendArgs {
  Batch b;
  Rot r;
  const void *k, *v, *q;
  void* q_out;
  long long k_ts, k_hs, v_ts, v_hs, q_ts, q_hs, o_ts, o_hs;
  int HQ, rows, row_groups;
};

template <int HD> constexpr int LANES_PER_ROW = HD <= 32 ? 4 : HD <= 64 ? 8 : 16;

// Rotates the 8 dims that this lane holds of a row.  Lanes of the row sit next
// to each other; `exch` (HD floats of the row) is used where a pair's other
// half is not a whole lane away.
template <int HD>
__device__ __forceinline__ void rotate8(float (&f)[8], int li, const float* row, int rot, bool inter, float* exch) {
  const int d0 = li * 8;
  if (inter) {
    #pragma unroll
    for (int i = 0; i < 4; ++i)
      if (d0 + 2 * i < rot) {
        const float2 cs = __ldg(reinterpret_cast<const float2*>(row) + d0 / 2 + i);
        turn(f[2 * i], f[2 * i + 1], cs.x, cs.y);
      }
    return;
  }
  const int half = rot >> 1;
  float o[8];                                            // the other elements of the pairs
  if ((half & 7) == 0) {
    const int up = half >> 3;
    const int lane = threadIdx.x & 31;
    const bool in = d0 < rot;
    const int src = !in ? lane : d0 < half ? lane + up : lane - up;
    #pragma unroll
    for (int i = 0; i < 8; ++i) o[i] = __shfl_sync(0xffffffffu, f[i], src);
    if (in) {
      const bool first = d0 < half;
      const float2* cs2 = reinterpret_cast<const float2*>(row) + (first ? d0 : d0 - half);
      #pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float2 cs = __ldg(cs2 + i);
        float a = first ? f[i] : o[i], b = first ? o[i] : f[i];
        turn(a, b, cs.x, cs.y);
        f[i] = first ? a : b;
      }
    }
  } else {
    #pragma unroll
    for (int i = 0; i < 8; ++i)
      if (d0 + i < HD) exch[d0 + i] = f[i];
    __syncwarp();
    #pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int d = d0 + i;
      if (d < rot) {
        const bool first = d < half;
        const int j = first ? d : d - half;
        const float2 cs = __ldg(reinterpret_cast<const float2*>(row) + j);
        float a = exch[j], b = exch[j + half];
        turn(a, b, cs.x, cs.y);
        f[i] = first ? a : b;
      }
    }
    __syncwarp();
  }
}

template <typename T, int HD, bool ALIGNED>
__global__ void __launch_bounds__(256) append_kernel(const AppendArgs a) {
  constexpr int LPR = LANES_PER_ROW<HD>, RPW = 32 / LPR, REC9 = HD * 9 / 8;
  __shared__ float s_exch[8][RPW][HD];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int li = lane % LPR, ri = lane / LPR;
  const long long wid = (long long)blockIdx.x * 8 + warp;
  const int t = (int)(wid / a.row_groups), rg = (int)(wid % a.row_groups);
  if (t >= a.b.T) return;
  const int seq = find_seq(a.b.q_start, a.b.n_seq, t);
  const int q_end = __ldg(a.b.q_start + seq + 1);
  const int pos = __ldg(a.b.lens + seq) - q_end + t;
  const bool held = t >= __ldg(a.b.q_start + seq) && t < q_end && pos >= 0 && (pos >> a.b.page_shift) < a.b.max_pages;
  const int pg = held ? __ldg(a.b.bt + (long long)seq * a.b.bt_ld + (pos >> a.b.page_shift)) : -1;
  const bool store = held && (unsigned)pg < (unsigned)a.b.n_pages;
  const float* row = nullptr;
  if (a.r.table) {
    const int p = a.r.positions ? __ldg(a.r.positions + t) : pos;
    row = a.r.table + (long long)min(max(p, 0), a.r.n_pos - 1) * a.r.rot;
  }
  const int slot = pos & (a.b.page - 1), page = a.b.page, H = a.b.H;
  #pragma unroll 1
  for (int k = 0; k < 4; ++k) {
    const int rw = (rg * 4 + k) * RPW + ri;                       // row of this token
    if ((rg * 4 + k) * RPW >= a.rows) break;
    const bool on = rw < a.rows && li * 8 < HD;
    const int what = rw < H ? 0 : rw < 2 * H ? 1 : 2;             // key, value, query
    const int h = rw - what * H;
    float f[8];
    #pragma unroll
    for (int i = 0; i < 8; ++i) f[i] = 0.f;
    if (on) {
      const T* p = what == 0 ? static_cast<const T*>(a.k) + t * a.k_ts + h * a.k_hs
                 : what == 1 ? static_cast<const T*>(a.v) + t * a.v_ts + h * a.v_hs
                             : static_cast<const T*>(a.q) + t * a.q_ts + h * a.q_hs;
      load_vec<T, 8, ALIGNED>(p + li * 8, f);
    }
    if (row) {
      float keep[8];
      #pragma unroll
      for (int i = 0; i < 8; ++i) keep[i] = f[i];
      rotate8<HD>(f, li, row, a.r.rot, a.r.inter, s_exch[warp][ri]);
      if (what == 1) {
        #pragma unroll
        for (int i = 0; i < 8; ++i) f[i] = keep[i];
      }
    }
    float top = 0.f;
    #pragma unroll
    for (int i = 0; i < 8; ++i) top = fmaxf(top, fabsf(f[i]));
    top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
    if (!on) continue;
    if (what == 2) {
      store_vec<T, 8, ALIGNED>(static_cast<T*>(a.q_out) + t * a.o_ts + h * a.o_hs + li * 8, f);
      continue;
    }
    if (!store) continue;
    const int e = tile_e(top);
    const float up = pow2f(3 - e);
    unsigned w = 0;
    #pragma unroll
    for (int i = 0; i < 8; ++i) w |= nibble(f[i], up) << (4 * i);
    uint8_t* rec = a.b.pool + ((long long)pg * H + h) * (page * REC9);
    if (what == 0) {
      *reinterpret_cast<unsigned*>(rec + ((slot >> 2) * (HD / 8) + li) * 16 + (slot & 3) * 4) = w;
    } else {
      uint8_t* vp = rec + page * HD / 2 + ((slot >> 3) * (HD / 4) + 2 * li) * 16 + (slot & 3) * 4 + (slot >> 2 & 1) * 2;
      *reinterpret_cast<uint16_t*>(vp) = (uint16_t)w;
      *reinterpret_cast<uint16_t*>(vp + 16) = (uint16_t)(w >> 16);
    }
    if ((li & 1) == 0) rec[page * HD + ((what * HD / 16) + li / 2) * page + slot] = (uint8_t)(e + 18);
  }
}

// ---------------------------------------------------------------------------
// read: 8 consecutive tokens of one head per warp, keys then values; a lane
// takes 8 dims of a token, so that the 8 tokens' bytes of one unit, which lie
// next to each other, are read together.
// ---------------------------------------------------------------------------
struct ReadArgs {
  Batch b;
  void *k, *v;          // [T][H][HD]
};

template <typename T, int HD>
__global__ void __launch_bounds__(256) read_kernel(const ReadArgs a) {
  constexpr int REC9 = HD * 9 / 8;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const long long wid = (long long)blockIdx.x * 8 + warp;
  const int H = a.b.H, page = a.b.page;
  const long long t0 = wid / H * 8;
  const int h = (int)(wid % H);
  if (t0 >= a.b.T) return;
  int seq = find_seq(a.b.q_start, a.b.n_seq, (int)t0);
  const long long t = t0 + (lane & 7);
  if (t >= a.b.T) return;
  while (seq + 1 < a.b.n_seq && __ldg(a.b.q_start + seq + 1) <= t) ++seq;
  const int q_end = __ldg(a.b.q_start + seq + 1);
  const int pos = __ldg(a.b.lens + seq) - q_end + (int)t;
  const bool held = t >= __ldg(a.b.q_start + seq) && t < q_end && pos >= 0 && (pos >> a.b.page_shift) < a.b.max_pages;
  const long long at = held ? record_of(a.b, seq, pos, h, page * REC9) : -1;
  const int slot = pos & (page - 1);
  const uint8_t* rec = a.b.pool + (at < 0 ? 0 : at);
  #pragma unroll
  for (int u = 0; u < HD / 8; u += 4) {
    const int un = u + (lane >> 3);                            // 8 dims
    unsigned kw = 0x88888888u, vw = 0x88888888u, ke = 21, ve = 21;
    if (at >= 0) {
      kw = __ldg(reinterpret_cast<const unsigned*>(rec + ((slot >> 2) * (HD / 8) + un) * 16 + (slot & 3) * 4));
      const uint8_t* vp = rec + page * HD / 2 + ((slot >> 3) * (HD / 4) + 2 * un) * 16 + (slot & 3) * 4 + (slot >> 2 & 1) * 2;
      vw = __ldg(reinterpret_cast<const unsigned short*>(vp)) |
           ((unsigned)__ldg(reinterpret_cast<const unsigned short*>(vp + 16)) << 16);
      ke = __ldg(rec + page * HD + (un >> 1) * page + slot);
      ve = __ldg(rec + page * HD + (HD / 16 + (un >> 1)) * page + slot);
    }
    const float ks = pow2f((int)ke - 21), vs = pow2f((int)ve - 21);
    float kf[8], vf[8];
    #pragma unroll
    for (int i = 0; i < 8; ++i) {
      kf[i] = (float)((int)(kw >> (4 * i) & 15u) - 8) * ks;
      vf[i] = (float)((int)(vw >> (4 * i) & 15u) - 8) * vs;
    }
    const long long o = (t * H + h) * HD + un * 8;
    store_vec<T, 8, true>(static_cast<T*>(a.k) + o, kf);
    store_vec<T, 8, true>(static_cast<T*>(a.v) + o, vf);
  }
}

template <typename T, int HD>
cudaError_t launch_append(AppendArgs a, bool aligned, cudaStream_t s) {
  constexpr int RPW = 32 / LANES_PER_ROW<HD>;
  a.row_groups = (a.rows + 4 * RPW - 1) / (4 * RPW);
  const long long blocks = ((long long)a.b.T * a.row_groups + 7) / 8;
  if (blocks > 0x7fffffffLL) return cudaErrorInvalidConfiguration;
  if (aligned) append_kernel<T, HD, true><<<(unsigned)blocks, 256, 0, s>>>(a);
  else append_kernel<T, HD, false><<<(unsigned)blocks, 256, 0, s>>>(a);
  return cudaGetLastError();
}

template <typename T, int HD>
cudaError_t launch_read(const ReadArgs& a, cudaStream_t s) {
  const long long blocks = (((long long)a.b.T + 7) / 8 * a.b.H + 7) / 8;
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
  }
  if (a.b.T == 0 || a.b.n_seq == 0) return BFP200_OK;
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
  a.rows = 2 * a.b.H + a.HQ;
  a.row_groups = 0;
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
  if (a.b.T == 0 || a.b.n_seq == 0) return BFP200_OK;
  if (!in->k_out_dev || !in->v_out_dev) return bad("null pointer");
  if ((reinterpret_cast<uintptr_t>(in->k_out_dev) | reinterpret_cast<uintptr_t>(in->v_out_dev)) & 15u)
    return bad("outputs must be 16-byte aligned");
  int n_sm = 0;
  if (int rc = device_ready(who, &n_sm)) return rc;
  a.k = in->k_out_dev; a.v = in->v_out_dev;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
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
