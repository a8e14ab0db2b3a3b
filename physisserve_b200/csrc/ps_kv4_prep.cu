// Appending to and reading from the paged 4-bit K/V cache (sm_100a).
//
// kv4_prep_kernel -- per token: RMSNorm(Q), RMSNorm(K), RoPE of both, rotated Q out, rotated K and
//   V quantised into their cache rows.  Everything happens in registers between one read of q, k, v
//   and one write of q' and the 4.5-bit rows.  A thread owns whole blocks of 16 elements (32 bytes
//   of bf16: one 256-bit load), so a block's scale needs no exchange between threads; its blocks sit
//   at the same 16 columns of its heads, so it reads one slice of the rotation tables.
//
//   Bound: HBM, 9.125 C bytes a token (C = heads * 128, kv_heads = heads, bf16), against 12 C of the
//   bf16 ring.  Measured: 12 480 tokens of 40 heads in 150 us, 60 % of the copy bandwidth: about 7 400
//   warp instructions a token at 0.6 a clock and scheduler are what the time goes to.
//
//   K's sum of squares is accumulated in fp64: squares are exact there, and so is the sum of a bf16 row
//   whose elements lie within about 2^11 of one another; of other rows, and of fp32 ones, the order
//   moves the last of 53 bits, and with it a rounding of the row's 1/sqrt to 24 bits once in some 2^28
//   rows.  So what is quantised does not depend on the order of the sum.  (An fp32 sum's last bit moves
//   one bf16 rounding in ~10^4 and with it now and then a 4-bit code, a quarter of the value.)  A bf16
//   number becomes a double by moving its bits, not by
//   the conversion unit.  Q's sum stays fp32: nothing that it moves is quantised.
//
// kv4_read_kernel -- rows back as bf16 or fp32: a thread expands 8 code bytes and a scale of K and
//   of V to 16 numbers each (one 256-bit store each in bf16).  Bound: HBM, mostly by the writes; 34 320
//   rows of 12 heads in 45.5 us, 92 % of the copy bandwidth.

#include <stdio.h>
#include <string.h>

#include "ps_kv4.cuh"

namespace ps {
namespace {

struct DevSeq4 {
  int64_t row0;
  int64_t table_row;
  int64_t ring_row;
  uint64_t hw_magic, gw_magic;
  int32_t hw, gw, frame_offset, ring_frames, ring_slot0, kind;
};

enum : int32_t { kQ = 1, kK = 2, kV = 4, kNormQ = 8, kNormK = 16, kPre = 32, kSink = 64 };
constexpr int32_t kFull = kQ | kK | kV | kNormQ | kNormK;  // the chunk prep: specialised

struct PParams {
  const void* q;
  const void* k;
  const void* v;
  const void* wq;
  const void* wk;
  const float* cos;
  const float* sin;
  void* q_out;
  void* k_pre;
  const void* k_sink;
  int64_t q_stride, k_stride, v_stride, q_out_stride, k_pre_stride, k_sink_stride;
  Kv4Dev cache;
  Kv4Scale k_scale, v_scale;
  int64_t page_bytes;  // of all heads
  float eps, cq, ck;   // row lengths of Q and K
  int32_t heads;
  int32_t tpt;         // threads per token (whole warps)
  int32_t hstep;       // heads between a thread's consecutive blocks = tpt / 8
  int32_t tokens_cta;  // tokens per CTA (1 unless a token is one warp)
  int32_t tp, thp;     // pairs of the frame axis, of the frame + row axes
  int32_t axes;        // PS_TABLE_AXES
  int32_t flags, w_f32, early, wide;
  int32_t n_seqs, total;
  int32_t cum[PS_MAX_SEQS + 1];
  DevSeq4 seq[PS_MAX_SEQS];
};
static_assert(sizeof(PParams) <= 8192, "kernel parameters too large");

constexpr int kMaxTpt = 320;      // threads per token: 40 heads a pass
// Blocks of a role that a thread holds at most (fp32 blocks take twice the registers).
constexpr int max_blocks(int dtype) { return dtype == PS_BF16 ? 5 : 3; }

// 32 bytes as one load / store where the rows allow it.
__device__ __forceinline__ void ld32(const void* p, uint32_t* w, bool wide) {
  if (wide) {
    asm volatile("ld.global.nc.L1::no_allocate.v8.b32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];"
                 : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3]), "=r"(w[4]), "=r"(w[5]), "=r"(w[6]), "=r"(w[7])
                 : "l"(p));
  } else {
    const uint4 a = ld_stream(p), b = ld_stream(static_cast<const char*>(p) + 16);
    w[0] = a.x; w[1] = a.y; w[2] = a.z; w[3] = a.w;
    w[4] = b.x; w[5] = b.y; w[6] = b.z; w[7] = b.w;
  }
}
__device__ __forceinline__ void st32(void* p, const uint32_t* w, bool wide) {
  if (wide) {
    asm volatile("st.global.v8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"l"(p), "r"(w[0]), "r"(w[1]), "r"(w[2]),
                 "r"(w[3]), "r"(w[4]), "r"(w[5]), "r"(w[6]), "r"(w[7])
                 : "memory");
  } else {
    st_vec(p, make_uint4(w[0], w[1], w[2], w[3]));
    st_vec(static_cast<char*>(p) + 16, make_uint4(w[4], w[5], w[6], w[7]));
  }
}

// A block of 16 elements as 32-bit words.
template <typename T> struct Block;
template <> struct Block<__nv_bfloat16> {
  static constexpr int kWords = 8;
  __device__ __forceinline__ static void load(const void* p, uint32_t* w, bool wide) { ld32(p, w, wide); }
  __device__ __forceinline__ static void store(void* p, const uint32_t* w, bool wide) { st32(p, w, wide); }
  __device__ __forceinline__ static f32x2 pair(const uint32_t* w, int j) {
    return f2_make(__uint_as_float(w[j] << 16), __uint_as_float(w[j] & 0xffff0000u));
  }
  __device__ __forceinline__ static void set(uint32_t* w, int j, float lo, float hi) {
    w[j] = Pairs16<__nv_bfloat16>::pack_pair(lo, hi);
  }
  __device__ __forceinline__ static f32x2 round(f32x2 v) { return Pairs16<__nv_bfloat16>::round(v); }
  // sum += x^2 in fp64.  A bf16's exponent and fraction bits moved to a double's high word, with the
  // exponent rebased (zero and subnormals read as up to 2^-126: their squares vanish beside eps).
  __device__ __forceinline__ static double add_squares(const uint32_t* w, double sum) {
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const double lo = __hiloint2double(static_cast<int>((w[j] & 0x7fffu) * 8192u + 0x38000000u), 0);
      const double hi = __hiloint2double(static_cast<int>(((w[j] & 0x7fff0000u) >> 3) + 0x38000000u), 0);
      sum = fma(lo, lo, sum);
      sum = fma(hi, hi, sum);
    }
    return sum;
  }
  __device__ __forceinline__ static bool has_nan(const uint32_t* w) {
    bool nan = false;
#pragma unroll
    for (int j = 0; j < 8; ++j) nan |= (w[j] & 0x7fffu) > 0x7f80u || (w[j] & 0x7fff0000u) > 0x7f800000u;
    return nan;
  }
};
template <> struct Block<float> {
  static constexpr int kWords = 16;
  __device__ __forceinline__ static void load(const void* p, uint32_t* w, bool wide) {
    ld32(p, w, wide);
    ld32(static_cast<const char*>(p) + 32, w + 8, wide);
  }
  __device__ __forceinline__ static void store(void* p, const uint32_t* w, bool wide) {
    st32(p, w, wide);
    st32(static_cast<char*>(p) + 32, w + 8, wide);
  }
  __device__ __forceinline__ static f32x2 pair(const uint32_t* w, int j) {
    return f2_make(__uint_as_float(w[2 * j]), __uint_as_float(w[2 * j + 1]));
  }
  __device__ __forceinline__ static void set(uint32_t* w, int j, float lo, float hi) {
    w[2 * j] = __float_as_uint(lo);
    w[2 * j + 1] = __float_as_uint(hi);
  }
  __device__ __forceinline__ static f32x2 round(f32x2 v) { return v; }
  __device__ __forceinline__ static double add_squares(const uint32_t* w, double sum) {
#pragma unroll
    for (int j = 0; j < 16; ++j) {
      const double x = __uint_as_float(w[j]);
      sum = fma(x, x, sum);
    }
    return sum;
  }
  __device__ __forceinline__ static bool has_nan(const uint32_t*) { return false; }  // the sum shows it
};

// 16 RMSNorm weights as pairs.
template <typename T>
__device__ __forceinline__ void weights16(const void* w, bool w_f32, int off, f32x2* out) {
  constexpr int E = Vec16<T>::kElems;
#pragma unroll
  for (int e = 0; e < 16; e += E) load_weight_pairs<T>(w, w_f32, off + e, out + e / 2);
}

// Quantises 16 numbers into the cache row at `codes` / `scale_byte`.
__device__ __forceinline__ void put_block(f32x2* x, const Kv4Scale& scale, unsigned char* codes,
                                          unsigned char* scale_byte) {
  float top = 0.f;
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    float a, b;
    f2_split(x[j], a, b);
    top = max3_abs(top, a, b);
  }
  const float most = 448.f * scale.six;  // the largest number the cache holds
  if (!(top <= most)) {                  // rare: NaN becomes 0, everything larger saturates
    if (!(top < INFINITY)) atomicAdd(&g_kv4_counts[kKv4NonFinite], 1u);
    top = 0.f;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      float v[2];
      f2_split(x[j], v[0], v[1]);
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        v[e] = isnan(v[e]) ? 0.f : fminf(fmaxf(v[e], -most), most);
        top = fmaxf(top, fabsf(v[e]));
      }
      x[j] = f2_make(v[0], v[1]);
    }
  }
  uint2 c;
  const uint32_t byte = kv4_quantise(x, top, scale, c);
  *reinterpret_cast<uint2*>(codes) = c;
  *scale_byte = static_cast<unsigned char>(byte);
}

// The roles one after another -- V, K, Q -- so that a thread holds the raw blocks of two roles at most (K's
// loads are in flight while V is quantised): registers, and with them the tokens an SM works on side by
// side, bound this kernel before memory does.
template <typename T, int NB, bool FULL>
__global__ void __launch_bounds__(NB == 5 ? 256 : kMaxTpt, NB == 5 ? 2 : 1) kv4_prep_kernel(const __grid_constant__ PParams p) {
  using B = Block<T>;
  constexpr int W = B::kWords;
  __shared__ double part_k[kMaxTpt / 32];
  __shared__ float part_q[kMaxTpt / 32];
  const int flags = FULL ? kFull : p.flags;
  const int slot = p.tokens_cta > 1 ? static_cast<int>(threadIdx.x) / p.tpt : 0;
  const int lt = static_cast<int>(threadIdx.x) - slot * p.tpt;
  const int slice = lt & 7, head0 = lt >> 3;
  const int g0 = blockIdx.x * p.tokens_cta + slot;
  const bool active = g0 < p.total;
  const int g = active ? g0 : 0;
  int lo = 0, hi = p.n_seqs - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (p.cum[mid] <= g) lo = mid; else hi = mid - 1;
  }
  const DevSeq4& sq = p.seq[lo];
  const int l = g - p.cum[lo];
  const int64_t row = sq.row0 + l;
  const bool sink = !FULL && (flags & kSink) && sq.kind == PS_SEQ_SINK;
  const bool do_q = (flags & kQ) && !sink, do_v = (flags & kV) && !sink, do_k = (flags & kK) || sink;
  const bool norm_q = (flags & kNormQ) && !sink, norm_k = (flags & kNormK) && !sink;
  const bool pre = !FULL && (flags & kPre) && !sink;
  // Head i of this thread, and its block's columns.
  const int col0 = head0 * kKv4D + slice * 16, col_step = p.hstep * kKv4D;
  auto has_q = [&](int i) { return head0 + i * p.hstep < p.heads; };
  auto has_k = [&](int i) { return head0 + i * p.hstep < p.cache.kv_heads; };

  if (!p.early) pdl_wait();
  uint32_t vw[NB][W], xw[NB][W];  // xw: K's blocks, then Q's
  if (active && do_v) {
    const T* src = static_cast<const T*>(p.v) + row * p.v_stride + col0;
#pragma unroll
    for (int i = 0; i < NB; ++i)
      if (has_k(i)) B::load(src + i * col_step, vw[i], p.wide);
  }
#pragma unroll
  for (int i = 0; i < NB; ++i)
#pragma unroll
    for (int j = 0; j < W; ++j) xw[i][j] = 0;
  if (active && do_k) {
    const T* src = (sink ? static_cast<const T*>(p.k_sink) + row * p.k_sink_stride
                         : static_cast<const T*>(p.k) + row * p.k_stride) + col0;
#pragma unroll
    for (int i = 0; i < NB; ++i)
      if (has_k(i)) B::load(src + i * col_step, xw[i], p.wide);
  }
  // Positions and the cache row.
  const int f = static_cast<int>(div_by(static_cast<uint32_t>(l), sq.hw_magic));
  const int rr = l - f * sq.hw;
  // (unsigned: a ring of one-token frames may have more than 2^30 of them)
  uint32_t ring = static_cast<uint32_t>(sq.ring_slot0) + static_cast<uint32_t>(f);
  if (ring >= static_cast<uint32_t>(sq.ring_frames)) ring -= static_cast<uint32_t>(sq.ring_frames);
  const int64_t kv_row = sq.ring_row + static_cast<int64_t>(ring) * sq.hw + rr;
  const int64_t page = active && (do_k || do_v) ? kv4_page(p.cache, kv_row >> p.cache.shift, lt == 0) : -1;
  // The token's K row of this thread's first head; V's is `half` bytes further, the next head's `step`.
  const int in_page = static_cast<int>(kv_row & ((1 << p.cache.shift) - 1));
  const int64_t half = p.cache.head_bytes >> 1, step = p.hstep * p.cache.head_bytes;
  unsigned char* const base = p.cache.pages + page * p.page_bytes + head0 * p.cache.head_bytes;
  const int code_off = in_page * 64 + slice * 8, scale_off = (64 << p.cache.shift) + in_page * 8 + slice;
  if (p.early) pdl_wait();
  if (do_v && page >= 0) {
#pragma unroll
    for (int i = 0; i < NB; ++i) {
      if (!has_k(i)) continue;
      f32x2 x[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) x[j] = B::pair(vw[i], j);
      unsigned char* const at = base + i * step + half;
      put_block(x, p.v_scale, at + code_off, at + scale_off);
    }
  }

  // This thread's slice of the rotation tables.
  f32x2 cc[8], ss[8];
  if (active && (do_q || do_k)) {
    int64_t t0, t1, t2;
    if (p.axes) {
      const int hh = static_cast<int>(div_by(static_cast<uint32_t>(rr), sq.gw_magic));
      t0 = sq.frame_offset + f;
      t1 = hh;
      t2 = rr - hh * sq.gw;
    } else {
      t0 = t1 = t2 = sq.table_row + l;
    }
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const int pair = slice * 8 + j;
      const int64_t at = (pair < p.tp ? t0 : (pair < p.thp ? t1 : t2)) * kKv4D + 2 * pair;
      cc[j] = __ldg(reinterpret_cast<const unsigned long long*>(p.cos + at));
      ss[j] = __ldg(reinterpret_cast<const unsigned long long*>(p.sin + at));
    }
  }

  // K.
  float rk = 1.f;
  if (flags & kNormK) {
    double sum = 0.0;
    if (norm_k) {
#pragma unroll
      for (int i = 0; i < NB; ++i)
        if (has_k(i)) sum = B::add_squares(xw[i], sum);
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    if (p.tpt > 32) {  // one token per CTA: every thread gets here
      if ((lt & 31) == 0) part_k[lt >> 5] = sum;
      __syncthreads();
      sum = 0.0;
      for (int i = 0; i < p.tpt >> 5; ++i) sum += part_k[i];
    }
    float ssq = static_cast<float>(sum);
    if (sizeof(T) == 2 && norm_k && isinf(ssq)) {  // uniform over the token: was there a NaN?
      bool nan = false;
#pragma unroll
      for (int i = 0; i < NB; ++i) nan |= B::has_nan(xw[i]);
      nan = p.tpt > 32 ? __syncthreads_or(nan) : __any_sync(0xffffffffu, nan);
      if (nan) ssq = NAN;
    }
    rk = rstd_of(ssq, p.ck, p.eps);
  }
  if (active && do_k) {
    const f32x2 r2 = f2_make(rk, rk);
#pragma unroll
    for (int i = 0; i < NB; ++i) {
      if (!has_k(i)) continue;
      const int off = col0 + i * col_step;
      f32x2 x[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) x[j] = B::pair(xw[i], j);
      if (norm_k) {
        f32x2 w[8];
        weights16<T>(p.wk, p.w_f32, off, w);
#pragma unroll
        for (int j = 0; j < 8; ++j) x[j] = B::round(f2_mul(f2_mul(x[j], r2), w[j]));
      }
      if (pre) {
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          float a, b;
          f2_split(x[j], a, b);
          B::set(xw[i], j, a, b);
        }
        B::store(static_cast<T*>(p.k_pre) + row * p.k_pre_stride + off, xw[i], p.wide);
      }
      if (page >= 0) {
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          float a, b;
          rotate_f2(x[j], cc[j], ss[j], a, b);
          x[j] = B::round(f2_make(a, b));  // what the ring would hold
        }
        unsigned char* const at = base + i * step;
        put_block(x, p.k_scale, at + code_off, at + scale_off);
      }
    }
  }

  // Q.
  if (!(flags & kQ)) {
    pdl_trigger();
    return;
  }
#pragma unroll
  for (int i = 0; i < NB; ++i)
#pragma unroll
    for (int j = 0; j < W; ++j) xw[i][j] = 0;
  if (active && do_q) {
    const T* src = static_cast<const T*>(p.q) + row * p.q_stride + col0;
#pragma unroll
    for (int i = 0; i < NB; ++i)
      if (has_q(i)) B::load(src + i * col_step, xw[i], p.wide);
  }
  pdl_trigger();  // every load is in flight: a dependent launch may be scheduled
  float rq = 1.f;
  if (flags & kNormQ) {
    f32x2 a = 0;
#pragma unroll
    for (int i = 0; i < NB; ++i)
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const f32x2 x = B::pair(xw[i], j);
        a = f2_fma(x, x, a);
      }
    float x, y;
    f2_split(a, x, y);
    float sum = x + y;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    if (p.tpt > 32) {
      if ((lt & 31) == 0) part_q[lt >> 5] = sum;
      __syncthreads();
      sum = 0.f;
      for (int i = 0; i < p.tpt >> 5; ++i) sum += part_q[i];
    }
    rq = rstd_of(sum, p.cq, p.eps);
  }
  if (!active || !do_q) return;
  const f32x2 r2 = f2_make(rq, rq);
  T* const dst = static_cast<T*>(p.q_out) + row * p.q_out_stride;
#pragma unroll
  for (int i = 0; i < NB; ++i) {
    if (!has_q(i)) continue;
    const int off = col0 + i * col_step;
    f32x2 w[8];
    if (norm_q) weights16<T>(p.wq, p.w_f32, off, w);
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      f32x2 x = B::pair(xw[i], j);
      if (norm_q) x = B::round(f2_mul(f2_mul(x, r2), w[j]));
      float a, b;
      rotate_f2(x, cc[j], ss[j], a, b);
      B::set(xw[i], j, a, b);
    }
    B::store(dst + off, xw[i], p.wide);
  }
}

// ---------------------------------------------------------------------------------------
// Reading rows
// ---------------------------------------------------------------------------------------
struct RParams {
  Kv4Dev cache;
  void* k_out;
  void* v_out;
  int64_t k_member, k_row, v_member, v_row;  // element strides
  int64_t row0;
  uint64_t rows_magic;   // div_magic(rows)
  uint32_t rows;
  uint32_t items;        // members * rows * kv_heads * 8
  uint64_t per_magic;    // div_magic(kv_heads * 8)
  uint32_t per;          // kv_heads * 8
  int32_t wide;
};

constexpr int kReadUnroll = 4;
constexpr int kReadThreads = 256;

template <typename T>
__device__ __forceinline__ void expand(uint2 codes, uint32_t byte, float tensor_scale, T* out, bool wide) {
  const uint32_t s2 = kv4_scales(byte | (byte << 8));
  uint32_t w[8];
  kv4_unpack(codes.x, w);
  kv4_unpack(codes.y, w + 4);
  uint32_t o[Block<T>::kWords];
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    const uint32_t h = h2_mul(w[j], s2);
    const float2 x = __half22float2(*reinterpret_cast<const __half2*>(&h));
    Block<T>::set(o, j, x.x * tensor_scale, x.y * tensor_scale);
  }
  Block<T>::store(out, o, wide);
}

template <typename T>
__global__ void __launch_bounds__(kReadThreads) kv4_read_kernel(const __grid_constant__ RParams p) {
  const uint32_t first = blockIdx.x * (kReadThreads * kReadUnroll) + threadIdx.x;
  uint2 kc[kReadUnroll], vc[kReadUnroll];
  uint32_t ks[kReadUnroll], vs[kReadUnroll], r[kReadUnroll], b[kReadUnroll], c[kReadUnroll];
  pdl_wait();
#pragma unroll
  for (int u = 0; u < kReadUnroll; ++u) {
    const uint32_t item = first + u * kReadThreads;
    kc[u] = vc[u] = make_uint2(0, 0);
    ks[u] = vs[u] = 0;
    if (item >= p.items) continue;
    const uint32_t flat = div_by(item, p.per_magic);
    c[u] = item - flat * p.per;
    b[u] = div_by(flat, p.rows_magic);
    r[u] = flat - b[u] * p.rows;
    const int64_t row = p.row0 + r[u];
    const int64_t page = kv4_page(p.cache, b[u] * p.cache.table_pages + (row >> p.cache.shift));
    if (page < 0) continue;
    const int in_page = static_cast<int>(row & ((1 << p.cache.shift) - 1));
    const unsigned char* base = kv4_head(p.cache, page, c[u] >> 3);
    const int64_t code = in_page * 64 + (c[u] & 7) * 8;
    const int64_t scale = (static_cast<int64_t>(64) << p.cache.shift) + in_page * 8 + (c[u] & 7);
    const int64_t half = p.cache.head_bytes >> 1;
    if (p.k_out) {
      kc[u] = *reinterpret_cast<const uint2*>(base + code);
      ks[u] = base[scale];
    }
    if (p.v_out) {
      vc[u] = *reinterpret_cast<const uint2*>(base + half + code);
      vs[u] = base[half + scale];
    }
  }
  pdl_trigger();
#pragma unroll
  for (int u = 0; u < kReadUnroll; ++u) {
    if (first + u * kReadThreads >= p.items) continue;
    if (p.k_out)
      expand(kc[u], ks[u], p.cache.k_scale,
             static_cast<T*>(p.k_out) + b[u] * p.k_member + r[u] * p.k_row + c[u] * 16, p.wide);
    if (p.v_out)
      expand(vc[u], vs[u], p.cache.v_scale,
             static_cast<T*>(p.v_out) + b[u] * p.v_member + r[u] * p.v_row + c[u] * 16, p.wide);
  }
}

// ---------------------------------------------------------------------------------------
// Host side
// ---------------------------------------------------------------------------------------
struct PPlan {
  PParams params;
  int dtype, nb, threads;
  int64_t blocks;
  bool pdl;
};

static int check16(const void* p, int64_t stride, int64_t C, int es, const char* name) {
  if (!p) return fail(PS_ERR_NULL, "%s is NULL", name);
  if (!aligned16(p)) return fail(PS_ERR_ALIGN, "%s is not 16-byte aligned", name);
  if (stride < C) return fail(PS_ERR_SHAPE, "%s row stride %lld is below its %lld columns", name, (long long)stride, (long long)C);
  if ((stride * es) % 16) return fail(PS_ERR_ALIGN, "%s row stride must be a multiple of 16 bytes", name);
  return PS_OK;
}
static bool wide32(const void* p, int64_t stride, int es) {
  return p == nullptr || ((reinterpret_cast<uintptr_t>(p) & 31u) == 0 && (stride * es) % 32 == 0);
}

// Blocks per thread and warps per token for the larger head count, by the instructions a token costs (counted
// on a B200, bf16): about 500 a warp (decode, tables, row sums) and 640 for a block of each of Q, K and V.
// 40 heads: five blocks and two warps 150 us, two blocks and five warps 162 us (12 480 tokens).
static void choose_split(int heads, int max_nb, int* nb, int* warps) {
  int best = 0;
  for (int n = 1; n <= max_nb; ++n) {
    const int w = (heads + 4 * n - 1) / (4 * n);
    const int cost = w * (500 + 640 * n);
    if (w * 32 <= kMaxTpt && (best == 0 || cost < best)) {
      best = cost;
      *nb = n;
      *warps = w;
    }
  }
}

// `sms`: of the device that the launch is for (its work split alone depends on it).
static int build_prep(const ps_kv4_prep_args* a, int sms, PPlan* plan) {
  clear_error();
  if (!a) return fail(PS_ERR_NULL, "args is NULL");
  if (a->dtype != PS_BF16 && a->dtype != PS_F32) return fail(PS_ERR_DTYPE, "dtype %d is not PS_BF16 or PS_F32", a->dtype);
  if (a->weight_f32 != 0 && a->weight_f32 != 1) return fail(PS_ERR_DTYPE, "weight_f32=%d is not 0 or 1", a->weight_f32);
  if (a->launch < PS_LAUNCH_STREAM || a->launch > PS_LAUNCH_PDL_EARLY_INPUTS)
    return fail(PS_ERR_SHAPE, "launch mode %d unknown", a->launch);
  if (a->head_dim != kKv4D) return fail(PS_ERR_UNSUPPORTED, "head_dim=%d: the 4-bit cache holds heads of 128", a->head_dim);
  if (a->n_seqs < 1) return fail(PS_ERR_SHAPE, "n_seqs=%d", a->n_seqs);
  if (a->n_seqs > PS_MAX_SEQS) return fail(PS_ERR_TOO_MANY_SEQS, "n_seqs=%d exceeds PS_MAX_SEQS=%d", a->n_seqs, PS_MAX_SEQS);
  if (!a->seqs) return fail(PS_ERR_NULL, "seqs is NULL");
  memset(plan, 0, sizeof(*plan));
  PParams& p = plan->params;
  int64_t cache_rows = 0;
  int rc = kv4_check_cache(a->cache, &p.cache, &cache_rows);
  if (rc) return rc;
  const int hk = a->cache.kv_heads;
  const int max_heads = a->dtype == PS_BF16 ? 120 : 80;
  if (a->heads < 1 || a->heads > max_heads || hk > max_heads)
    return fail(PS_ERR_UNSUPPORTED, "heads=%d kv_heads=%d: 1..%d", a->heads, hk, max_heads);
  const int es = a->dtype == PS_BF16 ? 2 : 4;
  const int64_t C = static_cast<int64_t>(a->heads) * kKv4D, Ck = static_cast<int64_t>(hk) * kKv4D;
  int sinks = 0;
  for (int s = 0; s < a->n_seqs; ++s) {
    if (a->seqs[s].kind != PS_SEQ_PREP && a->seqs[s].kind != PS_SEQ_SINK)
      return fail(PS_ERR_SHAPE, "seq %d: kind %d unknown", s, a->seqs[s].kind);
    sinks += a->seqs[s].kind == PS_SEQ_SINK;
  }
  const bool q = a->q, k = a->k, v = a->v;
  if (!q && !k && !v && !sinks) return fail(PS_ERR_NULL, "q, k and v are all NULL");
  if (a->q_weight && !q) return fail(PS_ERR_SHAPE, "q_weight given without q");
  if (a->k_weight && !k) return fail(PS_ERR_SHAPE, "k_weight given without k");
  if (a->k_pre && !k) return fail(PS_ERR_SHAPE, "k_pre given without k");
  const bool nq = a->q_weight, nk = a->k_weight;
  if ((nq || nk) && !(a->eps >= 0.f)) return fail(PS_ERR_SHAPE, "eps must be >= 0");
  p.wide = 1;
  if (q) {
    if ((rc = check16(a->q, a->q_stride, C, es, "q")) || (rc = check16(a->q_out, a->q_out_stride, C, es, "q_out"))) return rc;
    p.wide &= wide32(a->q, a->q_stride, es) && wide32(a->q_out, a->q_out_stride, es);
  }
  if (k && (rc = check16(a->k, a->k_stride, Ck, es, "k"))) return rc;
  if (v && (rc = check16(a->v, a->v_stride, Ck, es, "v"))) return rc;
  if (a->k_pre && (rc = check16(a->k_pre, a->k_pre_stride, Ck, es, "k_pre"))) return rc;
  p.wide &= (!k || wide32(a->k, a->k_stride, es)) && (!v || wide32(a->v, a->v_stride, es)) &&
            wide32(a->k_pre, a->k_pre_stride, es);
  if (sinks) {
    if ((rc = check16(a->k_sink, a->k_sink_stride, Ck, es, "k_sink"))) return rc;
    if (a->k_sink_rows < 0) return fail(PS_ERR_SHAPE, "k_sink_rows=%lld", (long long)a->k_sink_rows);
    p.wide &= wide32(a->k_sink, a->k_sink_stride, es);
  }
  if ((nq && !aligned16(a->q_weight)) || (nk && !aligned16(a->k_weight)))
    return fail(PS_ERR_ALIGN, "RMSNorm weights are not 16-byte aligned");
  const bool rotate = q || k || sinks;
  if (rotate) {
    if (!a->cos || !a->sin) return fail(PS_ERR_NULL, "cos or sin is NULL");
    if (!aligned16(a->cos) || !aligned16(a->sin)) return fail(PS_ERR_ALIGN, "cos or sin is not 16-byte aligned");
    if (a->table_rows < 1) return fail(PS_ERR_SHAPE, "table_rows=%lld", (long long)a->table_rows);
    if (a->table_mode != PS_TABLE_TOKENS && a->table_mode != PS_TABLE_AXES)
      return fail(PS_ERR_SHAPE, "table_mode %d unknown", a->table_mode);
    if (a->table_mode == PS_TABLE_AXES &&
        (a->t_dim < 0 || a->h_dim < 0 || a->w_dim < 0 || ((a->t_dim | a->h_dim | a->w_dim) & 1) ||
         a->t_dim + a->h_dim + a->w_dim != kKv4D))
      return fail(PS_ERR_SHAPE, "axis split %d/%d/%d must be even parts of 128", a->t_dim, a->h_dim, a->w_dim);
  }
  if (a->in_rows < 0) return fail(PS_ERR_SHAPE, "in_rows=%lld", (long long)a->in_rows);

  int64_t total = 0;
  for (int s = 0; s < a->n_seqs; ++s) {
    const ps_seq& sq = a->seqs[s];
    const bool sink = sq.kind == PS_SEQ_SINK;
    if (sq.n_tokens < 0 || sq.grid_h < 1 || sq.grid_w < 1)
      return fail(PS_ERR_SHAPE, "seq %d: n_tokens=%d grid=%dx%d", s, sq.n_tokens, sq.grid_h, sq.grid_w);
    const int64_t hw = static_cast<int64_t>(sq.grid_h) * sq.grid_w;
    if (hw > INT32_MAX || sq.n_tokens % hw)
      return fail(PS_ERR_SHAPE, "seq %d: n_tokens=%d is not whole frames of %lld tokens", s, sq.n_tokens, (long long)hw);
    const int64_t frames = sq.n_tokens / hw, src = sink ? a->k_sink_rows : a->in_rows;
    if (sq.n_tokens >= (1 << 30)) return fail(PS_ERR_UNSUPPORTED, "seq %d: sizes beyond 2^30 tokens", s);
    if (sq.token_start < 0 || sq.token_start > src - sq.n_tokens)
      return fail(PS_ERR_BOUNDS, "seq %d: rows [%lld, %lld) outside %s=%lld", s, (long long)sq.token_start,
                  (long long)(sq.token_start + sq.n_tokens), sink ? "k_sink_rows" : "in_rows", (long long)src);
    if (rotate && sq.n_tokens > 0) {
      if (a->table_mode == PS_TABLE_AXES) {
        if (sq.frame_offset < 0 || sq.frame_offset + frames > a->table_rows || sq.grid_h > a->table_rows ||
            sq.grid_w > a->table_rows)
          return fail(PS_ERR_BOUNDS, "seq %d: positions (frames %d..%lld, %dx%d) exceed table_rows=%lld", s,
                      sq.frame_offset, (long long)(sq.frame_offset + frames - 1), sq.grid_h, sq.grid_w,
                      (long long)a->table_rows);
      } else if (sq.table_row < 0 || sq.table_row > a->table_rows - sq.n_tokens) {
        return fail(PS_ERR_BOUNDS, "seq %d: table rows [%lld, %lld) exceed table_rows=%lld", s, (long long)sq.table_row,
                    (long long)(sq.table_row + sq.n_tokens), (long long)a->table_rows);
      }
    }
    if ((k || v || sink) && sq.n_tokens > 0) {
      if (sq.ring_frames < 1 || sq.ring_slot0 < 0 || sq.ring_slot0 >= sq.ring_frames)
        return fail(PS_ERR_BOUNDS, "seq %d: ring slot %d outside [0, %d)", s, sq.ring_slot0, sq.ring_frames);
      if (frames > sq.ring_frames)
        return fail(PS_ERR_BOUNDS, "seq %d: %lld frames would overwrite each other in a ring of %d", s, (long long)frames,
                    sq.ring_frames);
      if (sq.ring_row < 0 || sq.ring_row > cache_rows - static_cast<int64_t>(sq.ring_frames) * hw)
        return fail(PS_ERR_BOUNDS, "seq %d: ring rows [%lld, %lld) outside the cache's %lld", s, (long long)sq.ring_row,
                    (long long)(sq.ring_row + sq.ring_frames * hw), (long long)cache_rows);
    }
    p.cum[s] = static_cast<int32_t>(total);
    DevSeq4& d = p.seq[s];
    d.row0 = sq.token_start;
    d.table_row = sq.table_row;
    d.ring_row = sq.ring_row;
    d.hw_magic = div_magic(static_cast<uint32_t>(hw));
    d.gw_magic = div_magic(static_cast<uint32_t>(sq.grid_w));
    d.hw = static_cast<int32_t>(hw);
    d.gw = sq.grid_w;
    d.frame_offset = sq.frame_offset;
    d.ring_frames = sq.ring_frames > 0 ? sq.ring_frames : 1;
    d.ring_slot0 = sq.ring_slot0;
    d.kind = sq.kind;
    total += sq.n_tokens;
    if (total > (1 << 30)) return fail(PS_ERR_SHAPE, "more than 2^30 tokens in one call");
  }
  p.cum[a->n_seqs] = static_cast<int32_t>(total);
  p.total = static_cast<int32_t>(total);
  p.n_seqs = a->n_seqs;
  p.q = a->q; p.k = a->k; p.v = a->v; p.wq = a->q_weight; p.wk = a->k_weight;
  p.cos = a->cos; p.sin = a->sin; p.q_out = a->q_out; p.k_pre = a->k_pre; p.k_sink = a->k_sink;
  p.q_stride = a->q_stride; p.k_stride = a->k_stride; p.v_stride = a->v_stride;
  p.q_out_stride = a->q_out_stride; p.k_pre_stride = a->k_pre_stride; p.k_sink_stride = a->k_sink_stride;
  p.k_scale = kv4_scale_of(a->cache.k_scale);
  p.v_scale = kv4_scale_of(a->cache.v_scale);
  p.page_bytes = p.cache.head_bytes * hk;
  p.eps = a->eps;
  p.cq = static_cast<float>(C);
  p.ck = static_cast<float>(Ck);
  p.heads = a->heads;
  p.axes = a->table_mode == PS_TABLE_AXES;
  p.tp = p.axes ? a->t_dim / 2 : kKv4D;
  p.thp = p.axes ? (a->t_dim + a->h_dim) / 2 : kKv4D;
  p.flags = (q ? kQ : 0) | (k ? kK : 0) | (v ? kV : 0) | (nq ? kNormQ : 0) | (nk ? kNormK : 0) | (a->k_pre ? kPre : 0) |
            (sinks ? kSink : 0);
  p.w_f32 = a->dtype == PS_BF16 && a->weight_f32 == 1;
  p.early = a->launch == PS_LAUNCH_PDL_EARLY_INPUTS;
  plan->pdl = a->launch != PS_LAUNCH_STREAM;
  plan->dtype = a->dtype;
  int warps = 1;
  plan->nb = 1;
  // A launch whose tokens are all resident at once (18 warps an SM, at the 112 registers of two blocks a thread) is
  // bound by the time of a token, not by throughput: then one block a thread, or two of bf16, whichever come to fit
  // first.  8 tokens of 12 heads 3.2 us against 5.7, 800 tokens 6.0 against 7.5, 400 tokens of 40 heads 7.7 against
  // 10.7; past it 1 560 tokens of 12 heads 10.4 (one block) against 8.6.
  const int most = a->heads > hk ? a->heads : hk;
  choose_split(most, max_blocks(a->dtype), &plan->nb, &warps);
  const int64_t resident = 18ll * sms;
  for (int n = a->dtype == PS_BF16 ? 2 : 1; n >= 1; --n) {
    const int w = (most + 4 * n - 1) / (4 * n);
    if (n < plan->nb && w * 32 <= kMaxTpt && total * w <= resident) {
      plan->nb = n;
      warps = w;
    }
  }
  p.tpt = warps * 32;
  p.hstep = warps * 4;
  p.tokens_cta = warps == 1 ? 2 : 1;
  plan->threads = p.tpt * p.tokens_cta;
  plan->blocks = (total + p.tokens_cta - 1) / p.tokens_cta;
  return PS_OK;
}

template <typename P>
static cudaError_t launch_pdl(void (*fn)(P), const P& params, int64_t blocks, int threads, bool pdl, cudaStream_t stream) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(blocks));
  cfg.blockDim = dim3(threads);
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  if (pdl) {
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
  }
  return cudaLaunchKernelEx(&cfg, fn, params);
}

template <typename T, int NB>
static void (*prep_fn(bool full))(PParams) {
  return full ? kv4_prep_kernel<T, NB, true> : kv4_prep_kernel<T, NB, false>;
}
static void (*prep_fn(int dtype, int nb, bool full))(PParams) {
  if (dtype == PS_F32)
    return nb == 1 ? prep_fn<float, 1>(full) : nb == 2 ? prep_fn<float, 2>(full) : prep_fn<float, 3>(full);
  switch (nb) {
    case 1: return prep_fn<__nv_bfloat16, 1>(full);
    case 2: return prep_fn<__nv_bfloat16, 2>(full);
    case 3: return prep_fn<__nv_bfloat16, 3>(full);
    case 4: return prep_fn<__nv_bfloat16, 4>(full);
    default: return prep_fn<__nv_bfloat16, 5>(full);
  }
}

static int build_read(const ps_kv4_read_args* a, RParams* p) {
  clear_error();
  if (!a) return fail(PS_ERR_NULL, "args is NULL");
  if (a->dtype != PS_BF16 && a->dtype != PS_F32) return fail(PS_ERR_DTYPE, "dtype %d is not PS_BF16 or PS_F32", a->dtype);
  memset(p, 0, sizeof(*p));
  int64_t cache_rows = 0;
  int rc = kv4_check_cache(a->cache, &p->cache, &cache_rows);
  if (rc) return rc;
  const int es = a->dtype == PS_BF16 ? 2 : 4;
  const int64_t C = static_cast<int64_t>(a->cache.kv_heads) * kKv4D;
  const int64_t member_rows = a->cache.table_pages * a->cache.page_rows;
  if (a->row0 < 0 || a->rows < 0 || a->row0 > member_rows - a->rows)
    return fail(PS_ERR_BOUNDS, "rows [%lld, %lld) outside a member's %lld", (long long)a->row0,
                (long long)(a->row0 + a->rows), (long long)member_rows);
  if (!a->k_out && !a->v_out) return fail(PS_ERR_NULL, "k_out and v_out are both NULL");
  p->wide = 1;
  for (int i = 0; i < 2; ++i) {
    void* out = i ? a->v_out : a->k_out;
    const int64_t row = i ? a->v_row_stride : a->k_row_stride, member = i ? a->v_member_stride : a->k_member_stride;
    const char* name = i ? "v_out" : "k_out";
    if (!out) continue;
    if ((rc = check16(out, row, C, es, name))) return rc;
    if (a->cache.members > 1 && member < a->rows * row)
      return fail(PS_ERR_SHAPE, "%s member stride %lld overlaps %lld rows", name, (long long)member, (long long)a->rows);
    if ((member * es) % 16) return fail(PS_ERR_ALIGN, "%s member stride must be a multiple of 16 bytes", name);
    p->wide &= wide32(out, row, es) && (member * es) % 32 == 0;
  }
  const int64_t per = static_cast<int64_t>(a->cache.kv_heads) * 8;
  if (a->rows >= INT32_MAX || a->cache.members * a->rows > 0x7fffffffLL / per)
    return fail(PS_ERR_UNSUPPORTED, "%lld members of %lld rows in one read", (long long)a->cache.members, (long long)a->rows);
  p->k_out = a->k_out; p->v_out = a->v_out;
  p->k_member = a->k_member_stride; p->k_row = a->k_row_stride;
  p->v_member = a->v_member_stride; p->v_row = a->v_row_stride;
  p->row0 = a->row0;
  p->rows = static_cast<uint32_t>(a->rows);
  p->rows_magic = div_magic(p->rows);
  p->per = static_cast<uint32_t>(per);
  p->per_magic = div_magic(p->per);
  p->items = static_cast<uint32_t>(a->cache.members * a->rows * per);
  return PS_OK;
}

}  // namespace

int kv4_check_cache(const ps_kv4_cache& c, Kv4Dev* d, int64_t* rows) {
  if (!c.pages) return fail(PS_ERR_NULL, "pages is NULL");
  if (!c.table) return fail(PS_ERR_NULL, "table is NULL");
  if (!aligned16(c.pages)) return fail(PS_ERR_ALIGN, "pages is not 16-byte aligned");
  if (reinterpret_cast<uintptr_t>(c.table) & 3u) return fail(PS_ERR_ALIGN, "table is not 4-byte aligned");
  if (c.page_rows != 16 && c.page_rows != 32 && c.page_rows != 64 && c.page_rows != 128)
    return fail(PS_ERR_SHAPE, "page_rows=%d is not 16, 32, 64 or 128", c.page_rows);
  if (c.kv_heads < 1 || c.kv_heads > 4096) return fail(PS_ERR_SHAPE, "kv_heads=%d", c.kv_heads);
  if (c.num_pages < 1 || c.num_pages > INT32_MAX || c.members < 1 || c.members > (1 << 24) || c.table_pages < 1 ||
      c.table_pages > (1 << 26))
    return fail(PS_ERR_SHAPE, "num_pages=%lld members=%lld table_pages=%lld", (long long)c.num_pages,
                (long long)c.members, (long long)c.table_pages);
  // The scales within what keeps code * scale and its reciprocal far from fp32's ends.
  for (const float s : {c.k_scale, c.v_scale})
    if (!(s >= 1e-20f && s <= 1e20f)) return fail(PS_ERR_SHAPE, "tensor scale %g outside [1e-20, 1e20]", s);
  d->pages = static_cast<unsigned char*>(c.pages);
  d->table = c.table;
  d->table_pages = c.table_pages;
  d->head_bytes = 2ll * c.page_rows * kKv4Row;
  d->num_pages = static_cast<uint32_t>(c.num_pages);
  d->kv_heads = c.kv_heads;
  d->shift = c.page_rows == 16 ? 4 : c.page_rows == 32 ? 5 : c.page_rows == 64 ? 6 : 7;
  d->k_scale = c.k_scale;
  d->v_scale = c.v_scale;
  *rows = c.members * c.table_pages * c.page_rows;
  return PS_OK;
}

}  // namespace ps

extern "C" int32_t ps_kv4_prep_validate(const ps_kv4_prep_args* args) {
  ps::PPlan plan;
  return ps::build_prep(args, 148, &plan);
}

extern "C" int32_t ps_qk_norm_rope_kv4(const ps_kv4_prep_args* args, void* stream) {
  ps::PPlan plan;
  const int rc = ps::build_prep(args, ps::sm_count(), &plan);
  if (rc != PS_OK || plan.blocks == 0) return rc;
  const bool full = plan.params.flags == ps::kFull;
  auto fn = ps::prep_fn(plan.dtype, plan.nb, full);
  const cudaError_t err =
      ps::launch_pdl(fn, plan.params, plan.blocks, plan.threads, plan.pdl, static_cast<cudaStream_t>(stream));
  if (err != cudaSuccess) return ps::fail(PS_ERR_LAUNCH, "kv4 prep launch: %s", cudaGetErrorString(err));
  return PS_OK;
}

extern "C" int32_t ps_kv4_read_validate(const ps_kv4_read_args* args) {
  ps::RParams p;
  return ps::build_read(args, &p);
}

extern "C" int32_t ps_kv4_read(const ps_kv4_read_args* args, void* stream) {
  ps::RParams p;
  const int rc = ps::build_read(args, &p);
  if (rc != PS_OK || p.items == 0) return rc;
  const int64_t per = ps::kReadThreads * ps::kReadUnroll;
  const int64_t blocks = (static_cast<int64_t>(p.items) + per - 1) / per;
  auto fn = args->dtype == PS_BF16 ? ps::kv4_read_kernel<__nv_bfloat16> : ps::kv4_read_kernel<float>;
  const cudaError_t err = ps::launch_pdl(fn, p, blocks, ps::kReadThreads, true, static_cast<cudaStream_t>(stream));
  if (err != cudaSuccess) return ps::fail(PS_ERR_LAUNCH, "kv4 read launch: %s", cudaGetErrorString(err));
  return PS_OK;
}

extern "C" int32_t ps_kv4_counters(uint32_t* counts, int32_t reset) {
  ps::clear_error();
  if (!counts) return ps::fail(PS_ERR_NULL, "counts is NULL");
  counts[0] = counts[1] = counts[2] = 0;
  cudaError_t err = cudaDeviceSynchronize();
  if (err == cudaSuccess) err = ps::kv4_take_counts(counts, reset);
  if (err == cudaSuccess) err = ps::kv4_attention_counts(counts, reset);
  if (err != cudaSuccess) return ps::fail(PS_ERR_LAUNCH, "reading the cache counters: %s", cudaGetErrorString(err));
  return PS_OK;
}
