// The paged 4-bit K/V cache on the device: addressing, quantising and dequantising a block
// of 16 elements, the counters (format: include/physis_b200_kv4.h).
#pragma once

#include <cuda_fp16.h>

#include "physis_b200_kv4.h"
#include "ps_common.cuh"

namespace ps {

constexpr int kKv4D = PS_KV4_HEAD_DIM;
constexpr int kKv4Row = PS_KV4_ROW_BYTES;

// Counters of the translation unit that includes this header (ps_kv4_counters adds them up).
enum { kKv4BadPages, kKv4NonFinite, kKv4Timeouts, kKv4Counters };  // the timeouts last
static __device__ unsigned int g_kv4_counts[kKv4Counters];

// Adds this translation unit's counts to `counts` and clears those that `reset` (ps_kv4_reset) names.
static inline cudaError_t kv4_take_counts(uint32_t* counts, int reset) {
  uint32_t own[kKv4Counters] = {};
  cudaError_t err = cudaMemcpyFromSymbol(own, g_kv4_counts, sizeof(own));
  for (int i = 0; i < kKv4Counters; ++i) counts[i] += own[i];
  if (err == cudaSuccess && reset != PS_KV4_KEEP) {
    const int first = reset == PS_KV4_RESET_TIMEOUTS ? kKv4Timeouts : 0;
    memset(own, 0, sizeof(own));
    err = cudaMemcpyToSymbol(g_kv4_counts, own, (kKv4Counters - first) * sizeof(own[0]), first * sizeof(own[0]));
  }
  return err;
}
cudaError_t kv4_attention_counts(uint32_t* counts, int reset);  // ps_kv4_attention.cu

// SMs of the current device (of a B200 where there is none).
static inline int sm_count() {
  int dev = 0, n = 0;
  if (cudaGetDevice(&dev) == cudaSuccess && cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev) == cudaSuccess &&
      n > 0)
    return n;
  return 148;
}

// A cache as kernels see it.
struct Kv4Dev {
  unsigned char* pages;
  const int32_t* table;
  int64_t table_pages;   // entries per member
  int64_t head_bytes;    // K and V of one head in a page: 2 * page_rows * 72
  uint32_t num_pages;
  int32_t kv_heads;
  int32_t shift;         // log2(page_rows)
  float k_scale, v_scale;
};

// Validates `c` (host) and fills `d`; `rows` receives members * table_pages * page_rows.
int kv4_check_cache(const ps_kv4_cache& c, Kv4Dev* d, int64_t* rows);  // ps_kv4_prep.cu

// Page of a table entry's index, or -1 if the entry names no page of the pool (counted if `count`).
__device__ __forceinline__ int64_t kv4_page(const Kv4Dev& c, int64_t index, bool count = true) {
  const int32_t page = c.table[index];  // an ordinary load: the kernel before may have written it
  if (static_cast<uint32_t>(page) < c.num_pages) return page;
  if (count) atomicAdd(&g_kv4_counts[kKv4BadPages], 1u);
  return -1;
}

// First byte of (page, head): K codes, K scales, V codes, V scales.
__device__ __forceinline__ unsigned char* kv4_head(const Kv4Dev& c, int64_t page, int head) {
  return c.pages + (page * c.kv_heads + head) * c.head_bytes;
}

// ---------------------------------------------------------------------------------------
// Dequantising
// ---------------------------------------------------------------------------------------
// The four bytes of w as element pairs in fp16 (exact): out[i] = (low, high) four bits of byte i.
__device__ __forceinline__ void kv4_unpack(uint32_t w, uint32_t* out) {
  asm("{\n\t.reg .b8 b0, b1, b2, b3;\n\t"
      "mov.b32 {b0, b1, b2, b3}, %4;\n\t"
      "cvt.rn.f16x2.e2m1x2 %0, b0;\n\t"
      "cvt.rn.f16x2.e2m1x2 %1, b1;\n\t"
      "cvt.rn.f16x2.e2m1x2 %2, b2;\n\t"
      "cvt.rn.f16x2.e2m1x2 %3, b3;\n\t}"
      : "=r"(out[0]), "=r"(out[1]), "=r"(out[2]), "=r"(out[3])
      : "r"(w));
}
// Two e4m3 scales (low byte first) as an fp16 pair (exact).
__device__ __forceinline__ uint32_t kv4_scales(uint32_t two) {
  uint32_t r;
  asm("{\n\t.reg .b16 h;\n\tcvt.u16.u32 h, %1;\n\tcvt.rn.f16x2.e4m3x2 %0, h;\n\t}" : "=r"(r) : "r"(two));
  return r;
}
__device__ __forceinline__ uint32_t h2_mul(uint32_t a, uint32_t b) {
  uint32_t r;
  asm("mul.rn.f16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  return r;
}

// ---------------------------------------------------------------------------------------
// Quantising
// ---------------------------------------------------------------------------------------
// e4m3 byte of a non-negative number, to nearest even, saturating at 448.
__device__ __forceinline__ uint32_t e4m3_of(float x) {
  uint32_t r;
  asm("{\n\t.reg .b16 h;\n\tcvt.rn.satfinite.e4m3x2.f32 h, %1, %2;\n\tcvt.u32.u16 %0, h;\n\t}"
      : "=r"(r)
      : "f"(0.f), "f"(x));
  return r;
}
// Eight codes of four pairs: pair i in byte i, its first number in the low four bits.
__device__ __forceinline__ uint32_t e2m1_of(const f32x2* y) {
  uint32_t r;
  asm("{\n\t.reg .b8 b0, b1, b2, b3;\n\t.reg .f32 l, h;\n\t"
      "mov.b64 {l, h}, %1;\n\tcvt.rn.satfinite.e2m1x2.f32 b0, h, l;\n\t"
      "mov.b64 {l, h}, %2;\n\tcvt.rn.satfinite.e2m1x2.f32 b1, h, l;\n\t"
      "mov.b64 {l, h}, %3;\n\tcvt.rn.satfinite.e2m1x2.f32 b2, h, l;\n\t"
      "mov.b64 {l, h}, %4;\n\tcvt.rn.satfinite.e2m1x2.f32 b3, h, l;\n\t"
      "mov.b32 %0, {b0, b1, b2, b3};\n\t}"
      : "=r"(r)
      : "l"(y[0]), "l"(y[1]), "l"(y[2]), "l"(y[3]));
  return r;
}

// A tensor scale t as the quantisation uses it.
struct Kv4Scale {
  float t, six, inv_six;  // t, 6 t, 1 / (6 t)
};
static inline Kv4Scale kv4_scale_of(float t) { return Kv4Scale{t, 6.f * t, 1.f / (6.f * t)}; }

// Quantises 16 numbers x (8 pairs) whose largest magnitude is `top` (finite): the scale byte is
// returned, the codes go to `codes`.  Both formats have so few bits that numbers do lie midway
// between two of theirs, so both quotients, top / (6 t) and x / (scale t), have to be exact where they
// are representable: each is the product with a reciprocal, corrected once by its own remainder
// (Markstein's division, IBM J. Res. Dev. 34, 1990).  The remainder is exact, so a reciprocal that is
// an ulp or two off leaves 2^-44 of the quotient before its rounding.
__device__ __forceinline__ uint32_t kv4_quantise(const f32x2* x, float top, const Kv4Scale& scale, uint2& codes) {
  const float q0 = __fmul_rn(top, scale.inv_six);
  const uint32_t byte = e4m3_of(__fmaf_rn(__fmaf_rn(-q0, scale.six, top), scale.inv_six, q0));
  const uint32_t s2 = kv4_scales(byte);
  const float step = __fmul_rn(__half2float(__ushort_as_half(static_cast<unsigned short>(s2 & 0xffffu))), scale.t);
  float inv;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(inv) : "f"(step));
  inv = step > 0.f ? inv : 0.f;
  const f32x2 inv2 = f2_make(inv, inv), neg2 = f2_make(-step, -step);
  f32x2 y[8];
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    const f32x2 y0 = f2_mul(x[j], inv2);
    y[j] = f2_fma(f2_fma(y0, neg2, x[j]), inv2, y0);
  }
  codes = make_uint2(e2m1_of(y), e2m1_of(y + 4));
  return byte;
}

// max(|a|, |b|, |c|); NaN if one of them is.
__device__ __forceinline__ float max3_abs(float a, float b, float c) {
  float r;
  asm("max.NaN.abs.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}

}  // namespace ps
