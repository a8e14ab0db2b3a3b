// Attention over the paged 4-bit K/V cache (include/physis_b200_kv4.h), sm_100a.
//
// A K/V head's query rows are its (token, query head) pairs: row r = t * group + i is token t of
// query head kv_head * group + i, so query heads that share a K/V head share every byte read.

#include <math.h>
#include <stdio.h>
#include <string.h>

#include <mutex>
#include <type_traits>

#include "ps_kv4.cuh"
#include "ps_sm100.cuh"

namespace ps {
namespace {

constexpr int kTileKeys = 128;  // keys per tile: one page of the largest size
constexpr int kMaxChunks = 64;
constexpr int kTileBytes = kTileKeys * 2 * kKv4Row;

struct AParams {
  Kv4Dev cache;
  const __nv_bfloat16* q;
  __nv_bfloat16* out;
  const int32_t* lens;
  int64_t q_member, q_row, out_member, out_row;
  int32_t Lq, kv_max, causal_block, group;
  int32_t rows;          // query rows of a K/V head: Lq * group
  int32_t row_blocks;    // blocks of query rows per K/V head
  int32_t chunks;        // rows kernel: key chunks per unit; 0: by the members' lengths (plan_split)
  int32_t grid;          // tiles kernel: persistent CTAs
  int32_t min_steps;     // tiles kernel: fewest steps of a CTA
  int64_t units;         // members * kv_heads * row_blocks
  float scale_log2;      // softmax scale * k_scale * log2(e)
  float* ws_o;           // partial results: [slots][rows of a block][128] unnormalised sums (32-byte aligned in the
                         // tiles kernel, which stores 32 bytes at a time),
  float2* ws_ml;         // [slots][rows of a block] (reference in log2 units, sum); slots are
                         // [CTAs] (rows kernel) or [grid][2] (tiles kernel)
  int4* ws_units;        // tiles kernel: [units] (first CTA, last CTA, the first CTA's slot, 0);
                         // rows kernel without fixed chunks: [members] (Split::before, Split::chunks)
};

__device__ __forceinline__ bool wait_bar(uint32_t bar, uint32_t parity, volatile int* abort_flag, bool count = true) {
  return bar_wait_for(bar, parity, abort_flag, count, &g_kv4_counts[kKv4Timeouts]);
}

// The warp's wait: a test that does not block first (the phase has often completed already).
__device__ __forceinline__ bool warp_wait(uint32_t bar, uint32_t parity, volatile int* abort_flag, int lane) {
  if (__all_sync(0xffffffffu, bar_test(bar, parity))) return true;
  return __all_sync(0xffffffffu, wait_bar(bar, parity, abort_flag, lane == 0));
}

// Window rows of member b.
__device__ __forceinline__ int member_len(const AParams& p, int b) {
  if (!p.lens) return p.kv_max;
  const int n = p.lens[b];
  return n < 0 ? 0 : (n > p.kv_max ? p.kv_max : n);
}
// Keys that token t of a member with n window rows sees.
__device__ __forceinline__ int token_limit(const AParams& p, int n, int t) {
  if (p.causal_block == 0) return n;
  const int64_t lim = static_cast<int64_t>(n) - p.Lq + static_cast<int64_t>(t / p.causal_block + 1) * p.causal_block;
  return lim < 0 ? 0 : (lim > n ? n : static_cast<int>(lim));
}

// Probabilities are taken against a reference of their row, kLift (log2 units) below the largest score at the
// time that it was set; it is set anew only when a score exceeds it by more than kTop, so that it seldom moves.
// They reach 2^kTop then, and fp16 holds them from there (2^15 is its largest power of two) down to 2^-24: what is
// lost of one is at most 2^-32 of the largest probability.  With no lift keys below 2^-25 of it were dropped from
// P V but not from the sum, all of them together.  Both roundings are directed, so that kTop holds for scores
// whose steps are larger than 1 too.
constexpr float kLift = 7.f, kTop = 15.f;
__device__ __forceinline__ float reference_of(float top) { return __fadd_ru(top, -kLift); }
__device__ __forceinline__ float most_of(float reference) { return __fadd_rd(reference, kTop); }

// Power of two that brings a row's largest magnitude `top` (>= 0) into [1, 2), and its inverse; 1 for
// zero, subnormal and non-finite rows.  The inverse of 2^127 is subnormal: rows from there on come into
// [2, 4), which fp16 holds with the same bits.
__device__ __forceinline__ float row_power(float top, float& back) {
  uint32_t e = __float_as_uint(top) >> 23;
  if (e < 2 || e > 254) {
    back = 1.f;
    return 1.f;
  }
  e = min(e, 253u);
  back = __uint_as_float(e << 23);
  return __uint_as_float((254u - e) << 23);
}

// ---------------------------------------------------------------------------------------
// rows kernel: up to 8 query rows of a K/V head
// ---------------------------------------------------------------------------------------
// Bound: HBM, 144 bytes a (key, K/V head); measured 16 members x 1 row of 12 heads over 34 320 keys in 209
// to 225 us (on several B200s), 65 to 70 % of the copy bandwidth: a 128-key tile takes an SM 0.62 us where
// HBM takes 0.42, and what takes it is the dequantising (ncu: 0.58 instructions a clock and scheduler, ALU
// 48 %, tensor pipe 23 %, three CTAs' registers an SM).  One CTA takes a (member, K/V head, row block) and
// one chunk of its keys.  A producer warp brings 128-key tiles into a ring of shared-memory stages, one
// bulk copy per page (K and V of a head lie together in a page); four warps take 32 keys of a tile each.
// Both products run transposed on mma.m16n8k16 -- S^T = K Q^T and O^T = V^T P^T -- so that the
// keys and the head dimension fill the 16-row side and eight query rows the 8-column side: a single
// query row wastes 7/8 of an otherwise idle tensor pipe and no memory traffic, and a fragment of K or
// V is dequantised once whatever the number of rows.
//
// Fragments come straight from the packed bytes because the products' inner index may be permuted:
//  * S^T: lane (g, c) (g = lane / 4, c = lane % 4) reads 16 bytes, elements 32c .. 32c+31, of keys g
//    and g + 8; the m16n8k16 step s takes its bytes 2s and 2s+1.  Q's fragments are loaded by the same
//    rule.
//  * O^T: lane (g, c) needs elements 16g .. 16g+15 (one scale block) of four keys; the low nibbles of
//    two keys' bytes merged by a bit select are an fp16 pair along the keys after one conversion.
//  * the probabilities pass from S^T's accumulators to P^T's operand by movmatrix (8 x 8 transposes).
// Which key of an 8-row group sits at index i (key_of) is chosen so that both the 16-byte reads of K
// and the 8-byte reads of V spread over the shared-memory banks.
constexpr int kRowWarps = 4;
constexpr int kRowThreads = 32 * (kRowWarps + 1);
constexpr int kStages = 3;
constexpr int kBlockRows = 8;   // query rows of a CTA

__device__ __forceinline__ int key_of(int i) { return (0x65742130u >> (4 * i)) & 7; }  // 0 3 1 2 4 7 5 6

__device__ __forceinline__ void mma16816(float* d, const uint32_t* a, uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t transpose8(uint32_t x) {
  uint32_t r;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(x));
  return r;
}
__device__ __forceinline__ uint32_t h2_pack(float lo, float hi) {
  uint32_t r;
  asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}
__device__ __forceinline__ void bulk_load(uint32_t dst, const void* src, uint32_t bytes, uint32_t bar) {
  asm volatile(
      "cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(dst), "l"(src),
      "r"(bytes), "r"(bar)
      : "memory");
}

__device__ __forceinline__ float max3(float a, float b, float c) {
  float r;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}
__device__ __forceinline__ f32x2 f2_add(f32x2 a, f32x2 b) {
  f32x2 r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
// Waits for the tensor-memory loads issued so far, one of which filled r: nothing that reads r can be
// moved ahead of the wait.
__device__ __forceinline__ void tmem_wait_ld32(uint32_t* r) {
  asm volatile("tcgen05.wait::ld.sync.aligned;"
               : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7]),
                 "+r"(r[8]), "+r"(r[9]), "+r"(r[10]), "+r"(r[11]), "+r"(r[12]), "+r"(r[13]), "+r"(r[14]),
                 "+r"(r[15]), "+r"(r[16]), "+r"(r[17]), "+r"(r[18]), "+r"(r[19]), "+r"(r[20]), "+r"(r[21]),
                 "+r"(r[22]), "+r"(r[23]), "+r"(r[24]), "+r"(r[25]), "+r"(r[26]), "+r"(r[27]), "+r"(r[28]),
                 "+r"(r[29]), "+r"(r[30]), "+r"(r[31]));
}
__device__ __forceinline__ void tmem_wait_ld16(uint32_t* r) {
  asm volatile("tcgen05.wait::ld.sync.aligned;"
               : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7]),
                 "+r"(r[8]), "+r"(r[9]), "+r"(r[10]), "+r"(r[11]), "+r"(r[12]), "+r"(r[13]), "+r"(r[14]), "+r"(r[15]));
}
// 16 consecutive fp32 columns of this thread's TMEM lane.
__device__ __forceinline__ void tmem_ld16(uint32_t taddr, uint32_t* r) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 "
      "{%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
        "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
      : "r"(taddr));
}

// Which keys a CTA of the rows kernel takes.  The chunks of all members stand in a row, `before` of them ahead of
// this member's; each is kv_heads * row_blocks CTAs.  chunks == 0: the CTA has no work.
struct Split {
  int member, before, chunks;
};

struct RowsShared {
  alignas(128) unsigned char stage[kStages][kTileBytes];
  alignas(8) unsigned long long full[kStages], empty[kStages];
  uint32_t bad[kStages];  // bit s: segment (page) s of the tile is not in the pool
  int lim[kBlockRows];    // keys that each query row sees
  Split split;
  int abort;
};

// Members of unlike length get chunks of like length: the fewest tiles a chunk, out of four sizes between the mean
// and one that always fits, with which all chunks find a CTA of the grid.  By one warp.
constexpr int kMinChunkTiles = 2;  // fewest tiles of a chunk (12 heads over 1 716 keys: 10.1 us, with four 11.8)
__device__ __noinline__ Split plan_split(const AParams& p, int lane) {
  const int per = p.cache.kv_heads * p.row_blocks, members = static_cast<int>(p.units / per);
  const int room = static_cast<int>(gridDim.x) / per, at = static_cast<int>(blockIdx.x) / per;
  auto tiles_of = [&](int b) { return b < members ? (member_len(p, b) + kTileKeys - 1) / kTileKeys : 0; };
  int64_t sum = 0;
  int top = 0;
  for (int b = lane; b < members; b += 32) {
    const int t = tiles_of(b);
    sum += t;
    top = max(top, t);
  }
#pragma unroll
  for (int d = 16; d > 0; d >>= 1) {
    sum += __shfl_xor_sync(0xffffffffu, sum, d);
    top = max(top, __shfl_xor_sync(0xffffffffu, top, d));
  }
  const int low = max(max(kMinChunkTiles, (top + kMaxChunks - 1) / kMaxChunks), static_cast<int>((sum + room - 1) / room));
  // Sum of ceil(t / size) <= sum / size + members: with `high` everything fits.
  const int64_t fits = room > members ? (sum + room - members - 1) / (room - members) : top;
  const int high = max(low, static_cast<int>(min(fits, static_cast<int64_t>(top))));
  int size[4], need[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    size[i] = low + static_cast<int>(static_cast<int64_t>(high - low) * i / 4);
    need[i] = 0;
  }
  for (int b = lane; b < members; b += 32) {
    const int t = tiles_of(b);
#pragma unroll
    for (int i = 0; i < 4; ++i) need[i] += max(1, (t + size[i] - 1) / size[i]);
  }
  int chosen = high;
#pragma unroll
  for (int i = 3; i >= 0; --i)
    if (static_cast<int>(__reduce_add_sync(0xffffffffu, need[i])) <= room) chosen = size[i];
  int before = 0;
  for (int b0 = 0; b0 < members; b0 += 32) {
    const int own = b0 + lane < members ? max(1, (tiles_of(b0 + lane) + chosen - 1) / chosen) : 0;
    int upto = own;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const int x = __shfl_up_sync(0xffffffffu, upto, d);
      if (lane >= d) upto += x;
    }
    const unsigned past = __ballot_sync(0xffffffffu, at < before + upto);
    if (past) {
      const int l = __ffs(past) - 1;
      return Split{b0 + l, before + __shfl_sync(0xffffffffu, upto - own, l), __shfl_sync(0xffffffffu, own, l)};
    }
    before += __shfl_sync(0xffffffffu, upto, 31);
  }
  return Split{0, 0, 0};
}

__global__ void __launch_bounds__(kRowThreads, 3) kv4_rows_kernel(const __grid_constant__ AParams p) {
  constexpr int R = kBlockRows;
  extern __shared__ unsigned char smem_raw[];
  RowsShared& sh = *reinterpret_cast<RowsShared*>(
      reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(smem_raw) + 127) & ~uintptr_t(127)));
  volatile int* abort_flag = &sh.abort;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    for (int s = 0; s < kStages; ++s) {
      bar_init(saddr(&sh.full[s]), 1);
      bar_init(saddr(&sh.empty[s]), kRowWarps);
    }
    sh.abort = 0;
    if (p.chunks) {
      const int member = static_cast<int>(blockIdx.x / (static_cast<int64_t>(p.cache.kv_heads) * p.row_blocks * p.chunks));
      sh.split = Split{member, member * p.chunks, p.chunks};
    }
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (p.chunks == 0 && warp == 1) {
    pdl_wait();  // the lengths may come from the kernel before
    const Split split = plan_split(p, lane);
    if (lane == 0) sh.split = split;
  }
  __syncthreads();

  // The row blocks of a (member, head, chunk) are neighbours, so that the keys they share come from L2.
  const Split split = sh.split;
  if (split.chunks == 0) return;
  const int per = p.cache.kv_heads * p.row_blocks;
  int at = static_cast<int>(blockIdx.x - static_cast<int64_t>(split.before) * per);
  const int rb = at % p.row_blocks;
  at /= p.row_blocks;
  const int chunk = at % split.chunks, h = at / split.chunks, b = split.member;
  if (p.chunks == 0 && at == 0 && rb == 0 && threadIdx.x == 0)
    p.ws_units[b] = make_int4(split.before, split.chunks, 0, 0);
  pdl_wait();
  const int n = member_len(p, b);
  const int row0 = rb * R, row_end = min(row0 + R, p.rows);
  const int lim_low = token_limit(p, n, row0 / p.group);               // fewest keys of any row of the block
  const int lim_top = token_limit(p, n, (row_end - 1) / p.group);      // most keys
  const int tiles = (lim_top + kTileKeys - 1) / kTileKeys;
  const int j0 = static_cast<int>(static_cast<int64_t>(chunk) * tiles / split.chunks);
  const int j1 = static_cast<int>(static_cast<int64_t>(chunk + 1) * tiles / split.chunks);
  const int shift = p.cache.shift, page_rows = 1 << shift;
  const int segs = kTileKeys >> shift;  // pages per tile
  const uint32_t seg_bytes = static_cast<uint32_t>(p.cache.head_bytes);

  if (warp == kRowWarps) {
    // ------------------------------- producer -------------------------------
    int t = 0;
    if (lane < R) sh.lim[lane] = token_limit(p, n, min(row0 + lane, p.rows - 1) / p.group);
    __syncwarp();  // the consumers learn of all of them by lane 0's arrival below
    // Lane i: table entry of the tile's page i, a tile ahead (unconditional loads, so that nothing waits for
    // them before they are used).
    auto seen = [&](int j) { return lane < segs && j * kTileKeys + (lane << shift) < lim_top; };
    auto entry_of = [&](int j) {
      const int64_t i = seen(j) ? ((static_cast<int64_t>(j) * kTileKeys) >> shift) + lane : 0;
      uint32_t x;
      asm volatile("ld.global.u32 %0, [%1];" : "=r"(x) : "l"(p.cache.table + b * p.cache.table_pages + i));
      return x;
    };
    uint32_t entry = entry_of(j0);
    for (int j = j0; j < j1; ++j, ++t) {
      const int s = t % kStages;
      const bool mine = seen(j), valid_page = mine && entry < p.cache.num_pages;
      if (mine && !valid_page) atomicAdd(&g_kv4_counts[kKv4BadPages], 1u);
      const unsigned char* src = kv4_head(p.cache, valid_page ? entry : 0, h);
      entry = entry_of(j + 1);
      const unsigned valid = __ballot_sync(0xffffffffu, valid_page);
      const unsigned wanted = __ballot_sync(0xffffffffu, mine);
      if (t >= kStages && !warp_wait(saddr(&sh.empty[s]), ((t / kStages) & 1) ^ 1, abort_flag, lane)) break;
      const uint32_t bar = saddr(&sh.full[s]);
      if (lane == 0) {
        sh.bad[s] = wanted & ~valid;
        bar_expect_tx(bar, __popc(valid) * seg_bytes);
      }
      __syncwarp();
      if (valid_page) bulk_load(saddr(sh.stage[s]) + lane * seg_bytes, src, seg_bytes, bar);
    }
    pdl_trigger();
    // Every copy has landed before the CTA may exit (the consumers have waited for theirs unless the
    // CTA aborted).
    volatile int never = 0;
    for (int u = t > kStages ? t - kStages : 0; u < t; ++u)
      wait_bar(saddr(&sh.full[u % kStages]), (u / kStages) & 1, &never, lane == 0);
    __syncwarp();
  }

  // ------------------------------- consumers -------------------------------
  const int g = lane >> 2, c = lane & 3;
  float o[8][4];
  float m[2], l[2];
  {
#pragma unroll
    for (int t = 0; t < 8; ++t)
#pragma unroll
      for (int e = 0; e < 4; ++e) o[t][e] = 0.f;
    m[0] = m[1] = -INFINITY;
    l[0] = l[1] = 0.f;
  }
  if (warp < kRowWarps) {
    // Q: query row g of each group of eight, elements 32c .. 32c+31, scaled to fp16.
    uint32_t qf[16];
    float qs[2];   // score scale of the query rows 2c, 2c + 1
    {
      const int r = row0 + g;
      uint4 w[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) w[i] = make_uint4(0, 0, 0, 0);
      if (r < row_end) {
        const int t = r / p.group;
        const __nv_bfloat16* src =
            p.q + b * p.q_member + t * p.q_row + (h * p.group + (r - t * p.group)) * kKv4D + 32 * c;
#pragma unroll
        for (int i = 0; i < 4; ++i) w[i] = *reinterpret_cast<const uint4*>(src + 8 * i);
      }
      const uint32_t* v = reinterpret_cast<const uint32_t*>(w);
      uint32_t top = v[0] & 0x7fff7fffu;
#pragma unroll
      for (int i = 1; i < 16; ++i) top = __vmaxu2(top, v[i] & 0x7fff7fffu);
      top = max(top << 16, top & 0xffff0000u);
      top = max(top, __shfl_xor_sync(0xffffffffu, top, 1));
      top = max(top, __shfl_xor_sync(0xffffffffu, top, 2));
      float back;
      const float power = row_power(__uint_as_float(top), back);
#pragma unroll
      for (int i = 0; i < 16; ++i)
        qf[i] = h2_pack(__uint_as_float(v[i] << 16) * power, __uint_as_float(v[i] & 0xffff0000u) * power);
#pragma unroll
      for (int e = 0; e < 2; ++e) qs[e] = __shfl_sync(0xffffffffu, back, (2 * c + e) * 4) * p.scale_log2;
    }
    const int kg = key_of(g);                                   // K rows of this lane: kg, kg + 8
    const int v0 = key_of(2 * c), v1 = key_of(2 * c + 1);       // V rows: v0, v1, v0 + 8, v1 + 8
    const int k_codes = kg * 64 + c * 16, k_scale = page_rows * 64 + kg * 8 + c * 2;
    const int v_base = page_rows * kKv4Row;
    const int v_codes = v_base + g * 8, v_scale = v_base + page_rows * 64 + g;

    int s = 0, phase = 0;
    for (int j = j0; j < j1; ++j) {
      if (!warp_wait(saddr(&sh.full[s]), phase, abort_flag, lane)) break;
      const uint32_t bad = *reinterpret_cast<volatile uint32_t*>(&sh.bad[s]);
      const bool masked = (j + 1) * kTileKeys > lim_low || bad != 0;
      // This warp's 32 keys, two groups of 16 side by side: a group's products are chains of dependent MMAs,
      // and with few warps it is their latency that counts (one after the other: 16 x 1 rows over 34 320
      // keys 255 us instead of 214, with a fourth CTA an SM).
      constexpr int U = 2;
      const int key0 = warp * 32;
      float acc[U][4];
#pragma unroll
      for (int u = 0; u < U; ++u) {  // S^T
        const int key = key0 + 16 * u;
        const unsigned char* base = sh.stage[s] + (key >> shift) * seg_bytes;
        const int in0 = key & (page_rows - 1);
        const unsigned char* kc = base + in0 * 64 + k_codes;
        const unsigned char* ksc = base + in0 * 8 + k_scale;
        const uint4 w0 = *reinterpret_cast<const uint4*>(kc);
        const uint4 w1 = *reinterpret_cast<const uint4*>(kc + 8 * 64);
        const uint32_t s0 = kv4_scales(*reinterpret_cast<const uint16_t*>(ksc));
        const uint32_t s1 = kv4_scales(*reinterpret_cast<const uint16_t*>(ksc + 8 * 8));
        const uint32_t s0l = __byte_perm(s0, s0, 0x1010), s0h = __byte_perm(s0, s0, 0x3232);
        const uint32_t s1l = __byte_perm(s1, s1, 0x1010), s1h = __byte_perm(s1, s1, 0x3232);
        float part[4];  // the second half of the head dimension: a chain of its own
#pragma unroll
        for (int e = 0; e < 4; ++e) acc[u][e] = part[e] = 0.f;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          uint32_t x0[4], x1[4];
          kv4_unpack(i == 0 ? w0.x : i == 1 ? w0.y : i == 2 ? w0.z : w0.w, x0);
          kv4_unpack(i == 0 ? w1.x : i == 1 ? w1.y : i == 2 ? w1.z : w1.w, x1);
          const uint32_t sa = i < 2 ? s0l : s0h, sb = i < 2 ? s1l : s1h;
#pragma unroll
          for (int k = 0; k < 2; ++k) {
            const uint32_t a[4] = {h2_mul(x0[2 * k], sa), h2_mul(x1[2 * k], sb), h2_mul(x0[2 * k + 1], sa),
                                   h2_mul(x1[2 * k + 1], sb)};
            mma16816(k ? part : acc[u], a, qf[4 * i + 2 * k], qf[4 * i + 2 * k + 1]);
          }
        }
#pragma unroll
        for (int e = 0; e < 4; ++e) acc[u][e] = (acc[u][e] + part[e]) * qs[e & 1];
      }
      // Scores in log2 units; what a row does not see becomes -inf.
      if (masked) {
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const int lim = *const_cast<volatile int*>(&sh.lim[2 * c + e]) - j * kTileKeys;
#pragma unroll
          for (int u = 0; u < U; ++u)
#pragma unroll
            for (int k = 0; k < 2; ++k) {
              const int in_tile = key0 + 16 * u + kg + 8 * k;
              if (in_tile >= lim || ((bad >> (in_tile >> shift)) & 1)) acc[u][e + 2 * k] = -INFINITY;
            }
        }
      }
      bool grow = false;
      {
        const float most[2] = {most_of(m[0]), most_of(m[1])};
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
          for (int e = 0; e < 4; ++e) grow |= acc[u][e] > most[e & 1];
      }
      if (__any_sync(0xffffffffu, grow)) {
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          float top = -INFINITY;
#pragma unroll
          for (int u = 0; u < U; ++u) top = fmaxf(top, fmaxf(acc[u][e], acc[u][e + 2]));
          top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 4));
          top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 8));
          top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 16));
          const float next = fmaxf(m[e], reference_of(top));
          const float alpha = next == -INFINITY ? 1.f : fast_exp2(m[e] - next);
          m[e] = next;
          l[e] *= alpha;
#pragma unroll
          for (int q = 0; q < 8; ++q) {
            o[q][e] *= alpha;
            o[q][e + 2] *= alpha;
          }
        }
      }
      uint32_t pb[U][2];
      {
        const float r0 = m[0] == -INFINITY ? 0.f : m[0], r1 = m[1] == -INFINITY ? 0.f : m[1];
#pragma unroll
        for (int u = 0; u < U; ++u) {
          const float p0 = fast_exp2(acc[u][0] - r0), p1 = fast_exp2(acc[u][1] - r1);
          const float p2 = fast_exp2(acc[u][2] - r0), p3 = fast_exp2(acc[u][3] - r1);
          l[0] += p0 + p2;
          l[1] += p1 + p3;
          pb[u][0] = transpose8(h2_pack(p0, p1));
          pb[u][1] = transpose8(h2_pack(p2, p3));
        }
      }
      // O^T += V^T P^T.
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int key = key0 + 16 * u;
        const unsigned char* base = sh.stage[s] + (key >> shift) * seg_bytes;
        const int in0 = key & (page_rows - 1);
        uint2 w[4];
        uint32_t sc[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int r = in0 + (i & 1 ? v1 : v0) + (i >> 1) * 8;
          w[i] = *reinterpret_cast<const uint2*>(base + v_codes + r * 64);
          sc[i] = base[v_scale + r * 8];
        }
        if (masked) {  // rows that no query row sees and rows of a missing page hold anything: 0 * code = 0
        const int lim_top = *const_cast<volatile int*>(&sh.lim[R - 1]);
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const int in_tile = key + (i & 1 ? v1 : v0) + (i >> 1) * 8;
            if (j * kTileKeys + in_tile >= lim_top || ((bad >> (in_tile >> shift)) & 1)) sc[i] = 0;
          }
        }
        const uint32_t sa = kv4_scales(sc[0] | (sc[1] << 8)), sb = kv4_scales(sc[2] | (sc[3] << 8));
#pragma unroll
        for (int half = 0; half < 2; ++half) {
          const uint32_t a0 = half ? w[0].y : w[0].x, a1 = half ? w[1].y : w[1].x;
          const uint32_t b0 = half ? w[2].y : w[2].x, b1 = half ? w[3].y : w[3].x;
          constexpr uint32_t kLow = 0x0f0f0f0fu;
          uint32_t al[4], ah[4], bl[4], bh[4];
          kv4_unpack((a0 & kLow) | ((a1 << 4) & ~kLow), al);
          kv4_unpack(((a0 >> 4) & kLow) | (a1 & ~kLow), ah);
          kv4_unpack((b0 & kLow) | ((b1 << 4) & ~kLow), bl);
          kv4_unpack(((b0 >> 4) & kLow) | (b1 & ~kLow), bh);
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const uint32_t a[4] = {h2_mul(al[i], sa), h2_mul(ah[i], sa), h2_mul(bl[i], sb), h2_mul(bh[i], sb)};
            mma16816(o[half * 4 + i], a, pb[u][0], pb[u][1]);
          }
        }
      }
      __syncwarp();
      if (lane == 0) bar_arrive(saddr(&sh.empty[s]));
      if (++s == kStages) {
        s = 0;
        phase ^= 1;
      }
    }
    // The rows' sums over the lanes that share them.
#pragma unroll
    for (int e = 0; e < 2; ++e)
#pragma unroll
      for (int d = 4; d < 32; d <<= 1) l[e] += __shfl_xor_sync(0xffffffffu, l[e], d);
  }
  // The four warps' results meet in the stages' memory: no copy is in flight any more.
  __syncthreads();
  constexpr int kStride = kKv4D + 4;
  float* part = reinterpret_cast<float*>(sh.stage);                        // [warp][R][kStride]
  float2* stat = reinterpret_cast<float2*>(part + kRowWarps * R * kStride);  // [warp][R]
  static_assert((kRowWarps * R * kStride + 2 * kRowWarps * R) * 4 <= kStages * kTileBytes, "merge buffer");
  if (warp < kRowWarps) {
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const int r = 2 * c + e;
      float* dst = part + (warp * R + r) * kStride + 16 * g;
#pragma unroll
      for (int q = 0; q < 8; q += 2)
        *reinterpret_cast<float4*>(dst + 2 * q) =
            make_float4(o[q][e], o[q][e + 2], o[q + 1][e], o[q + 1][e + 2]);
      if (g == 0) stat[warp * R + r] = make_float2(m[e], l[e]);
    }
  }
  __syncthreads();
  if (warp == kRowWarps) return;
  // Where the rows go: decoded once more, so that nothing of it stays in registers over the keys.
  const volatile Split& own = sh.split;
  const int chunks = own.chunks, member = own.member;
  const int in_member = static_cast<int>(blockIdx.x - static_cast<int64_t>(own.before) * p.cache.kv_heads * p.row_blocks);
  const int first_row = in_member % p.row_blocks * R, head = in_member / p.row_blocks / chunks;
  for (int r = warp; r < min(R, p.rows - first_row); r += kRowWarps) {
    float top = -INFINITY, sum = 0.f;
#pragma unroll
    for (int w = 0; w < kRowWarps; ++w) top = fmaxf(top, stat[w * R + r].x);
    float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
    for (int w = 0; w < kRowWarps; ++w) {
      const float2 ml = stat[w * R + r];
      // A warp that saw nothing has a zero sum; a NaN score leaves its reference at -inf and a NaN sum.
      const float f = ml.x == top || ml.y == 0.f ? (ml.y == 0.f ? 0.f : 1.f) : fast_exp2(ml.x - top);
      const float4 y = *reinterpret_cast<const float4*>(part + (w * R + r) * kStride + 4 * lane);
      if (ml.y == 0.f) continue;
      sum += f * ml.y;
      x.x += f * y.x;
      x.y += f * y.y;
      x.z += f * y.z;
      x.w += f * y.w;
    }
    if (chunks > 1) {
      const int64_t slot = static_cast<int64_t>(blockIdx.x) * R + r;
      *reinterpret_cast<float4*>(p.ws_o + slot * kKv4D + 4 * lane) = x;
      if (lane == 0) p.ws_ml[slot] = make_float2(top, sum);
    } else {
      const float inv = sum == 0.f ? 0.f : p.cache.v_scale / sum;
      const int row = first_row + r, t = row / p.group;
      __nv_bfloat16* dst =
          p.out + member * p.out_member + t * p.out_row + (head * p.group + (row - t * p.group)) * kKv4D + 4 * lane;
      *reinterpret_cast<uint2*>(dst) = make_uint2(Pairs16<__nv_bfloat16>::pack_pair(x.x * inv, x.y * inv),
                                                  Pairs16<__nv_bfloat16>::pack_pair(x.z * inv, x.w * inv));
    }
  }
}

// Merges the key chunks of a query row: out = v_scale * sum_c 2^(m_c - m) O_c / sum_c 2^(m_c - m) l_c.
// A warp per row.
__global__ void __launch_bounds__(128) kv4_combine_kernel(const __grid_constant__ AParams p) {
  constexpr int R = kBlockRows;
  const int lane = threadIdx.x & 31;
  const int64_t at = static_cast<int64_t>(blockIdx.x) * 4 + (threadIdx.x >> 5);
  const int64_t bh = at / p.rows;  // (member, K/V head)
  if (bh >= p.units / p.row_blocks) return;
  const int row = static_cast<int>(at - bh * p.rows);
  const int b = static_cast<int>(bh / p.cache.kv_heads), h = static_cast<int>(bh % p.cache.kv_heads);
  const int rb = row / R;
  pdl_wait();
  int before = b * p.chunks, chunks = p.chunks;
  if (chunks == 0) {
    const int4 info = p.ws_units[b];
    before = info.x;
    chunks = info.y;
    if (chunks == 1) return;  // the rows kernel wrote the row
  }
  const int64_t first = static_cast<int64_t>(before) * p.cache.kv_heads + static_cast<int64_t>(h) * chunks;
  const int64_t slot0 = (first * p.row_blocks + rb) * R + (row - rb * R), step = static_cast<int64_t>(p.row_blocks) * R;
  float top = -INFINITY;
  float2 ml[2];
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int ch = lane + 32 * i;
    ml[i] = ch < chunks ? p.ws_ml[slot0 + ch * step] : make_float2(-INFINITY, 0.f);
    top = fmaxf(top, ml[i].x);
  }
#pragma unroll
  for (int d = 16; d > 0; d >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, d));
  float f[2], sum = 0.f;
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    f[i] = ml[i].y == 0.f ? 0.f : (ml[i].x == top ? 1.f : fast_exp2(ml[i].x - top));
    sum += f[i] * ml[i].y;
  }
#pragma unroll
  for (int d = 16; d > 0; d >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, d);
  float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
  const float* src = p.ws_o + slot0 * kKv4D + 4 * lane;
  // 16 chunks at a time, so that their loads are in flight together.
  for (int c0 = 0; c0 < chunks; c0 += 16) {
    float4 y[16];
#pragma unroll
    for (int i = 0; i < 16; ++i)
      y[i] = *reinterpret_cast<const float4*>(src + min(c0 + i, chunks - 1) * step * kKv4D);
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      const float w = __shfl_sync(0xffffffffu, c0 < 32 ? f[0] : f[1], (c0 + i) & 31);
      if (w == 0.f) continue;  // behind the last chunk, or a chunk in which the row saw nothing
      x.x += w * y[i].x;
      x.y += w * y[i].y;
      x.z += w * y[i].z;
      x.w += w * y[i].w;
    }
  }
  const float inv = sum == 0.f ? 0.f : p.cache.v_scale / sum;
  const int t = row / p.group;
  __nv_bfloat16* dst = p.out + b * p.out_member + t * p.out_row + (h * p.group + (row - t * p.group)) * kKv4D + 4 * lane;
  *reinterpret_cast<uint2*>(dst) = make_uint2(Pairs16<__nv_bfloat16>::pack_pair(x.x * inv, x.y * inv),
                                              Pairs16<__nv_bfloat16>::pack_pair(x.z * inv, x.w * inv));
}

// ---------------------------------------------------------------------------------------
// tiles kernel: 256 query rows of a K/V head at a time, tcgen05
// ---------------------------------------------------------------------------------------
// Bound: the tensor cores (4 * 128 * 256 flops a key), with the 16 exponentials a clock of an SM's
// special-function unit next (256 of them a key: as many clocks as the products take).  Measured: 1 560
// rows of 12 heads over 34 320 keys in 388 to 396 us, 830 to 848 TFLOP/s, half of the library's bf16 rate; a step of two
// query tiles takes 4 350 clocks, the products 2 048 of them, the exponentials 2 275 when both tiles'
// warps run them.  What is left is their waiting for one another.
//
// A unit is (member, K/V head, 256 query rows) = two 128-row query tiles that share every K/V tile.
// Its work is the 128-key tiles that any of its rows sees ("steps").  The steps of all units, in
// order, are cut into equal contiguous ranges, one per CTA, one CTA per SM: every SM gets the same
// number of steps whatever the windows' lengths and masks are, and at most the first and the last unit
// of a range are shared with a neighbour.  Those leave partial results (unnormalised O, reference,
// sum) in two workspace slots per CTA; kv4_merge_kernel joins them.
//
// CTA of four warpgroups:
//   warp 14      brings the packed K and V of the tiles (9 KB each) into a ring of three shared-memory slots,
//                one bulk copy per page;
//   warps 0-3    dequantise: fp16 tiles in the 128-byte swizzled layout that the tensor core reads, two of K
//                and two of V;
//   warps 4-7    softmax of query tile 0, warps 8-11 of tile 1: a query row per thread (TMEM lane = row);
//                they also bring the row's Q, scaled to fp16, into shared memory.  The two warps of an SM
//                sub-partition take turns at exponentiating: side by side they would wait for the products
//                side by side too, and the special-function unit and the tensor core would idle in turn
//                instead of overlapping;
//   warps 12, 13 one thread each issues the MMAs of query tile 0 / 1, in the order PV(t), S(t+1): two
//                issuers, so that neither tile's products wait behind the other's softmax, and the time
//                between two issues of one (descriptors, barrier tests) is filled by the other's.  P
//                overwrites the S columns that were read; P V starts on the first half of the keys while
//                the second half is exponentiated.  Warp 12 owns the tensor memory (512 columns:
//                O0 | S0 | O1 | S1).
//   warp 15      writes which CTAs share each unit, for the merge.
// tcgen05.mma operations of one thread complete in issue order, so a commit after S_i(t+1) also reports
// P_i(t) V(t) done.  All waits are bounded: one that runs out raises the CTA's abort flag, every role
// leaves its loop, the issuers wait for their MMAs and the tensor memory is freed; the rows' values are
// undefined then, the units' table is not.
constexpr int kM = 128;
constexpr int kUnitRows = 2 * kM;
constexpr int kTile16 = kM * kKv4D * 2;    // bytes of a 128 x 128 fp16 tile
constexpr int kHalf16 = kTile16 / 2;       // its 64-column half
constexpr int kRawBytes = kTileKeys * kKv4Row;  // a packed tile of K or V
constexpr int kRawSlots = 3;
constexpr int kTilesThreads = 512;
constexpr int kOffQ = 0, kOffK = kOffQ + 2 * kTile16, kOffV = kOffK + 2 * kTile16, kOffRaw = kOffV + 2 * kTile16;
constexpr int kOffBars = kOffRaw + kRawSlots * kRawBytes;
enum TBar {
  kQFull, kKFull = kQFull + 2, kKEmpty = kKFull + 2, kVFull = kKEmpty + 2, kVEmpty = kVFull + 2, kSFull = kVEmpty + 2,
  kPHalf = kSFull + 2, kPFull = kPHalf + 2, kOFinal = kPFull + 2, kRawFull = kOFinal + 2, kRawEmpty = kRawFull + kRawSlots,
  kTurn = kRawEmpty + kRawSlots, kMmaDone = kTurn + 8, kTBars
};
constexpr int kOffTmem = kOffBars + 8 * kTBars, kOffAbort = kOffTmem + 4, kOffThere = kOffAbort + 4;
constexpr int kOffStart = (kOffThere + 4 * kRawSlots + 15) & ~15;
constexpr int kOffFactor = kOffStart + 32;  // [256] the factor of a row's scores in tensor memory
constexpr int kTilesSmem = kOffFactor + 4 * kUnitRows + 1024;
static_assert(kTilesSmem <= 227 * 1024, "tiles exceed shared memory");
// The softmax fuses a score's scaling with the taking off of its row's reference.  The reference is made of scores
// scaled and rounded, and from 2^24 on the product that is not rounded may lie further from it than fp16's range
// above kTop has room for.  A row whose reference gets beyond kNear has its scores scaled, and so rounded, in
// tensor memory from then on.  (Rounding every product in the softmax itself: 1.3B block call 385 -> 392 us; this
// costs 391 -> 392.5.)
constexpr float kNear = 0x1p22f;
__host__ __device__ constexpr int col_o(int i) { return 256 * i; }
__host__ __device__ constexpr int col_s(int i) { return 256 * i + 128; }
// kind::f16 with fp16 operands, fp32 accumulators, M = N = 128; b_mn: B's N runs along its rows.
__host__ __device__ constexpr uint32_t idesc16(uint32_t b_mn) {
  return (1u << 4) | (b_mn << 16) | ((128u >> 3) << 17) | ((128u >> 4) << 24);
}

// One K = 16 step of S = Q K^T: both operands OFFSET bytes into their tiles.  The descriptor's address
// field holds address >> 4 and shared addresses stay below 2^18, so the sum cannot carry out of it.
// Everything is formed inside the statement: descriptors of all steps kept in registers do not fit the
// issuing warp's share, and a spilled one costs more than the tensor core has queued.
template <int OFFSET>
__device__ __forceinline__ void mma_ss(uint32_t d, uint32_t a_low, uint32_t b_low, uint32_t high, bool acc) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t.reg .b32 a, b;\n\t.reg .b64 x, y;\n\t"
      "add.u32 a, %1, %6;\n\tadd.u32 b, %2, %6;\n\t"
      "mov.b64 x, {a, %3};\n\tmov.b64 y, {b, %3};\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], x, y, %5, p;\n\t}" ::"r"(d),
      "r"(a_low), "r"(b_low), "r"(high), "r"(acc ? 1u : 0u), "n"(idesc16(0)), "n"(OFFSET >> 4)
      : "memory");
}
// Step STEP (16 keys) of O += P V: P from tensor memory (8 columns a step), V's key rows 2 KB a step.
template <int STEP>
__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t a, uint32_t b_low, uint32_t high, bool acc) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t.reg .b32 a, b;\n\t.reg .b64 y;\n\t"
      "add.u32 a, %1, %6;\n\tadd.u32 b, %2, %7;\n\t"
      "mov.b64 y, {b, %3};\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [a], y, %5, p;\n\t}" ::"r"(d),
      "r"(a), "r"(b_low), "r"(high), "r"(acc ? 1u : 0u), "n"(idesc16(1)), "n"(STEP * 8), "n"(STEP * 128)
      : "memory");
}

// wait_bar inline (a call costs its registers).  Nearly every wait ends within a few suspended tries; only
// then is the clock read (it is slow).
__device__ __forceinline__ bool spin_bar(uint32_t bar, uint32_t parity, volatile int* abort_flag) {
  if (bar_test(bar, parity)) return true;
#pragma unroll 1
  for (int i = 0; i < 64; ++i)
    if (bar_try(bar, parity)) return true;
  const unsigned long long start = now_ns();
  for (;;) {
#pragma unroll 1
    for (int i = 0; i < 32; ++i)
      if (bar_try(bar, parity)) return true;
    if (*abort_flag) return false;
    if (now_ns() - start > kBarWaitNs) {
      atomicAdd(&g_kv4_counts[kKv4Timeouts], 1u);
      *abort_flag = 1;
      return false;
    }
  }
}
__device__ __forceinline__ bool warp_spin(uint32_t bar, uint32_t parity, volatile int* abort_flag) {
  return __all_sync(0xffffffffu, spin_bar(bar, parity, abort_flag));
}

// The scores of this thread's TMEM lane times f.
__device__ __noinline__ void scale_scores(uint32_t s_addr, float f) {
#pragma unroll 1
  for (int col = 0; col < 128; col += 16) {
    uint32_t y[16];
    tmem_ld16(s_addr + col, y);
    tmem_wait_ld16(y);
#pragma unroll
    for (int i = 0; i < 16; ++i) y[i] = __float_as_uint(__uint_as_float(y[i]) * f);
    tmem_st16(s_addr + col, y);
  }
  tmem_wait_st();
}

// Steps of a unit of member b with n window rows: the 128-key tiles that any of its rows sees, at least
// one (a unit that sees nothing still has zeros to write).
__device__ __forceinline__ int unit_steps(const AParams& p, int n, int qb, int& lim_top) {
  const int last = min((qb + 1) * kUnitRows, p.rows) - 1;
  lim_top = token_limit(p, n, last / p.group);
  return max(1, (lim_top + kTileKeys - 1) / kTileKeys);
}

// A CTA's way through its range of `count` steps; every role walks the same way.
struct Walk {
  int b, h, qb, lim_top;
  int j0, j1;        // key tiles of the present segment
  int steps;         // steps of the present unit
  int done, count;   // steps before the present segment, steps of the CTA

  __device__ __forceinline__ bool begin(const AParams& p, const int4& start, int n_steps) {
    b = start.x;
    h = start.y;
    qb = start.z;
    j0 = start.w;
    done = 0;
    count = n_steps;
    if (count == 0) return false;
    open(p);
    return true;
  }
  __device__ __forceinline__ void open(const AParams& p) {
    steps = unit_steps(p, member_len(p, b), qb, lim_top);
    j1 = min(steps, j0 + (count - done));
  }
  __device__ __forceinline__ bool next(const AParams& p) {
    done += j1 - j0;
    if (done >= count) return false;
    j0 = 0;
    if (++qb == p.row_blocks) {
      qb = 0;
      if (++h == p.cache.kv_heads) {
        h = 0;
        ++b;
      }
    }
    open(p);
    return true;
  }
  __device__ __forceinline__ bool first() const { return done == 0; }  // the CTA's first segment
  __device__ __forceinline__ bool two(const AParams& p) const { return qb * kUnitRows + kM < p.rows; }
  __device__ __forceinline__ bool whole() const { return j0 == 0 && j1 == steps; }
  __device__ __forceinline__ int64_t unit(const AParams& p) const {
    return (static_cast<int64_t>(b) * p.cache.kv_heads + h) * p.row_blocks + qb;
  }
};

// Total steps, and the unit and tile at which step `per * cta` lies (one warp; `per` is derived from the
// total).
__device__ __forceinline__ void find_start(const AParams& p, int64_t members, int lane, int64_t& per, int64_t& total,
                                           int4& start) {
  int lim;
  const int hk = p.cache.kv_heads;
  if (!p.lens && p.causal_block == 0) {  // every unit has the same number of steps
    const int steps = unit_steps(p, p.kv_max, 0, lim);
    total = p.units * steps;
    per = max((total + p.grid - 1) / p.grid, static_cast<int64_t>(p.min_steps));
    const int64_t u = per * blockIdx.x / steps;
    const int64_t bh = u / p.row_blocks;
    start = make_int4(static_cast<int>(bh / hk), static_cast<int>(bh % hk), static_cast<int>(u % p.row_blocks),
                      static_cast<int>(per * blockIdx.x % steps));
    return;
  }
  auto member_steps = [&](int b) {
    const int n = member_len(p, b);
    int64_t sum = 0;
    for (int q = lane; q < p.row_blocks; q += 32) sum += unit_steps(p, n, q, lim);
#pragma unroll
    for (int d = 16; d > 0; d >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, d);
    return sum;
  };
  total = 0;
  for (int b = 0; b < members; ++b) total += hk * member_steps(b);
  per = max((total + p.grid - 1) / p.grid, static_cast<int64_t>(p.min_steps));
  int64_t left = per * blockIdx.x;
  start = make_int4(0, 0, 0, 0);
  if (left >= total) return;
  int b = 0;
  int64_t sum = member_steps(0);
  while (left >= hk * sum) {
    left -= hk * sum;
    sum = member_steps(++b);
  }
  const int h = static_cast<int>(left / sum);
  left -= h * sum;
  const int n = member_len(p, b);
  for (int q0 = 0;; q0 += 32) {
    const int mine = q0 + lane < p.row_blocks ? unit_steps(p, n, q0 + lane, lim) : 0;
    int64_t upto = mine;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const int64_t y = __shfl_up_sync(0xffffffffu, upto, d);
      if (lane >= d) upto += y;
    }
    const unsigned past = __ballot_sync(0xffffffffu, upto > left);
    if (past) {
      const int l = __ffs(past) - 1;
      const int64_t before = __shfl_sync(0xffffffffu, upto - mine, l);
      start = make_int4(b, h, q0 + l, static_cast<int>(left - before));
      return;
    }
    left -= __shfl_sync(0xffffffffu, upto, 31);
  }
}

__global__ void __launch_bounds__(kTilesThreads, 1)
    kv4_tiles_kernel(const __grid_constant__ AParams p, const int64_t members) {
  extern __shared__ unsigned char smem_raw[];
  unsigned char* smem = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  const uint32_t sbase = saddr(smem);
  auto bar = [&](int i) { return sbase + kOffBars + 8u * static_cast<uint32_t>(i); };
  volatile int* abort_flag = reinterpret_cast<volatile int*>(smem + kOffAbort);
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(smem + kOffTmem);
  int64_t* range = reinterpret_cast<int64_t*>(smem + kOffStart);  // [per, total], then the start
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

  if (threadIdx.x == 0) {
    for (int i = 0; i < 2; ++i) {
      bar_init(bar(kQFull + i), 4);
      bar_init(bar(kKFull + i), 4);
      bar_init(bar(kKEmpty + i), 2);   // both issuers
      bar_init(bar(kVFull + i), 4);
      bar_init(bar(kVEmpty + i), 2);
      bar_init(bar(kSFull + i), 1);
      bar_init(bar(kPHalf + i), 4);
      bar_init(bar(kPFull + i), 4);
      bar_init(bar(kOFinal + i), 1);
    }
    for (int i = 0; i < kRawSlots; ++i) {
      bar_init(bar(kRawFull + i), 1);
      bar_init(bar(kRawEmpty + i), 4);
    }
    for (int i = 0; i < 8; ++i) bar_init(bar(kTurn + i), 1);
    bar_init(bar(kMmaDone), 2);
    *abort_flag = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 12) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(saddr(tmem_slot)), "r"(512)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  pdl_wait();
  if (warp == 0) {
    int64_t per, total;
    int4 start;
    find_start(p, members, lane, per, total, start);
    if (lane == 0) {
      range[0] = per;
      range[1] = total;
      *reinterpret_cast<int4*>(range + 2) = start;
    }
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  const int64_t per = range[0];
  const int4 start = *reinterpret_cast<int4*>(range + 2);
  const int n_steps = static_cast<int>(max(min(per, range[1] - per * blockIdx.x), int64_t(0)));
  const int shift = p.cache.shift;
  Walk w;

  if (warp < 4) {
    // ------------------------------- dequantisers -------------------------------
    // Lane (r, c): 16-byte chunk c (elements 32c .. 32c+31) of keys 32 i + 8 warp + r, i = 0..3.  Chunks 0
    // and 1 go to the fp16 tile's left half, 2 and 3 to its right one, whose rows fall into the same
    // banks: lanes of the right half take their four 8-element parts in the order 2 3 0 1, so that eight
    // lanes of a store cover all banks.
    const int r = lane >> 2, c = lane & 3;
    const bool right = c >= 2;
    const int page_rows = 1 << shift;
    // Byte offset of part 0 (in write order) of key row 8 warp + r; part i is at dst0 ^ (16 i).
    const uint32_t dst0 = (c >> 1) * kHalf16 + (8 * warp + r) * 128 + ((((c & 1) * 4) ^ (right ? 2 : 0) ^ r) * 16);
    const uint32_t sel_a = right ? 0x3232 : 0x1010, sel_b = right ? 0x1010 : 0x3232;
    uint32_t from[4];  // of key i: offsets of its code chunk (low half) and scale pair (high half) in a slot
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int key = 32 * i + 8 * warp + r, in_page = key & (page_rows - 1);
      const uint32_t seg = (key >> shift) * (page_rows * kKv4Row);
      from[i] = (seg + in_page * 64 + c * 16 + (right ? 8 : 0)) | ((seg + page_rows * 64 + in_page * 8 + c * 2) << 16);
    }
    const uint32_t every_page = (1u << (kTileKeys >> shift)) - 1;
    int t = 0, slot = 0;
    uint32_t slot_phase = 0;
    bool ok = true;
    for (bool more = w.begin(p, start, n_steps); ok && more; more = w.next(p)) {
      for (int j = w.j0; ok && j < w.j1; ++j, ++t) {
        const int st = t & 1;
        // K, then V (one copy of the code for both: see the softmax loops).
#pragma unroll 1
        for (int kv = 0; kv < 2; ++kv) {
          if (!(ok = warp_spin(bar(kRawFull + slot), slot_phase, abort_flag))) break;
          if (t >= 2 && !(ok = warp_spin(bar((kv ? kVEmpty : kKEmpty) + st), ((t >> 1) & 1) ^ 1, abort_flag))) break;
          const uint32_t raw = sbase + kOffRaw + slot * kRawBytes;
          const uint32_t tile = sbase + (kv ? kOffV : kOffK) + st * kTile16;
          uint32_t x[4][4], s2[4];
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const uint32_t src = raw + (from[i] & 0xffffu);
            asm volatile("ld.shared.v2.b32 {%0,%1}, [%2];" : "=r"(x[i][0]), "=r"(x[i][1]) : "r"(src));
            asm volatile("ld.shared.v2.b32 {%0,%1}, [%2];" : "=r"(x[i][2]), "=r"(x[i][3]) : "r"(src ^ 8));
            uint16_t two;
            asm volatile("ld.shared.u16 %0, [%1];" : "=h"(two) : "r"(raw + (from[i] >> 16)));
            s2[i] = two;
          }
          const uint32_t there = *reinterpret_cast<volatile uint32_t*>(smem + kOffThere + 4 * slot);
          const int seen = w.lim_top - j * kTileKeys;
          // What a missing or unseen key holds must not reach the products, even times a probability of 0.
          if (seen < kTileKeys || there != every_page) {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              const int key = 32 * i + 8 * warp + r;
              if (key >= seen || !((there >> (key >> shift)) & 1)) s2[i] = 0;
            }
          }
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const uint32_t sc = kv4_scales(s2[i]);
            const uint32_t sa = __byte_perm(sc, sc, sel_a), sb = __byte_perm(sc, sc, sel_b);
#pragma unroll
            for (int k = 0; k < 4; ++k) {
              uint32_t o[4];
              kv4_unpack(x[i][k], o);
              const uint32_t f = k < 2 ? sa : sb;
              asm volatile("st.shared.v4.b32 [%0], {%1,%2,%3,%4};" ::"r"(tile + (dst0 ^ (16 * k)) + 32 * i * 128),
                           "r"(h2_mul(o[0], f)), "r"(h2_mul(o[1], f)), "r"(h2_mul(o[2], f)), "r"(h2_mul(o[3], f))
                           : "memory");
            }
          }
          asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
          __syncwarp();
          if (lane == 0) {
            bar_arrive(bar(kRawEmpty + slot));
            bar_arrive(bar((kv ? kVFull : kKFull) + st));
          }
          if (++slot == kRawSlots) {
            slot = 0;
            slot_phase ^= 1;
          }
        }
      }
    }
  } else if (warp >= 12) {
    if (warp == 14) {
      // ------------------------------- bulk copies -------------------------------
      const uint32_t bytes = static_cast<uint32_t>(p.cache.head_bytes >> 1);  // K or V of a head in a page
      const int per_tile = kTileKeys >> shift;
      int u = 0;
      bool ok = true;
      for (bool more = w.begin(p, start, n_steps); ok && more; more = w.next(p)) {
        // Lane i: table entry of the tile's page i, a tile ahead.
        auto entry_of = [&](int j) {
          int32_t x = -1;
          if (lane < per_tile && j < w.j1 && j * kTileKeys + (lane << shift) < w.lim_top)
            x = p.cache.table[w.b * p.cache.table_pages + ((j * kTileKeys) >> shift) + lane];
          return x;
        };
        int32_t entry = entry_of(w.j0);
        for (int j = w.j0; ok && j < w.j1; ++j) {
          const bool wanted = lane < per_tile && j * kTileKeys + (lane << shift) < w.lim_top;
          const bool valid = wanted && static_cast<uint32_t>(entry) < p.cache.num_pages;
          if (wanted && !valid) atomicAdd(&g_kv4_counts[kKv4BadPages], 1u);
          const uint32_t there = __ballot_sync(0xffffffffu, valid);
          const unsigned char* src = kv4_head(p.cache, valid ? entry : 0, w.h);
          entry = entry_of(j + 1);
#pragma unroll
          for (int kv = 0; kv < 2; ++kv, ++u) {
            const int slot = u % kRawSlots;
            if (u >= kRawSlots && !(ok = warp_spin(bar(kRawEmpty + slot), ((u / kRawSlots) & 1) ^ 1, abort_flag))) break;
            if (lane == 0) {
              *reinterpret_cast<volatile uint32_t*>(smem + kOffThere + 4 * slot) = there;
              bar_expect_tx(bar(kRawFull + slot), __popc(there) * bytes);
            }
            __syncwarp();
            if (valid)
              bulk_load(sbase + kOffRaw + slot * kRawBytes + lane * bytes, src + kv * bytes, bytes, bar(kRawFull + slot));
          }
        }
      }
      // Every copy has landed before the CTA may exit.
      volatile int never = 0;
      for (int x = u > kRawSlots ? u - kRawSlots : 0; x < u; ++x)
        spin_bar(bar(kRawFull + x % kRawSlots), (x / kRawSlots) & 1, &never);
      __syncwarp();
    } else if (warp < 14 && lane == 0) {
      // ------------------------------- MMA issuers -------------------------------
      const int i = warp - 12;
      // Low words of the descriptors (address and leading byte offset); the high word is the same for all.
      const uint64_t q_desc = smem_desc(sbase + kOffQ + i * kTile16, 16, 1024);
      const uint32_t high = static_cast<uint32_t>(q_desc >> 32), q_low = static_cast<uint32_t>(q_desc);
      const uint32_t k_low = static_cast<uint32_t>(smem_desc(sbase + kOffK, 16, 1024));
      const uint32_t v_low = static_cast<uint32_t>(smem_desc(sbase + kOffV, kHalf16, 1024));
      const uint32_t s_col = tmem + col_s(i), o_col = tmem + col_o(i);
      auto issue_s = [&](int t) {
        const uint32_t k = k_low + ((t & 1) ? kTile16 >> 4 : 0);
        mma_ss<0>(s_col, q_low, k, high, false);
        mma_ss<32>(s_col, q_low, k, high, true);
        mma_ss<64>(s_col, q_low, k, high, true);
        mma_ss<96>(s_col, q_low, k, high, true);
        mma_ss<kHalf16>(s_col, q_low, k, high, true);
        mma_ss<kHalf16 + 32>(s_col, q_low, k, high, true);
        mma_ss<kHalf16 + 64>(s_col, q_low, k, high, true);
        mma_ss<kHalf16 + 96>(s_col, q_low, k, high, true);
      };
      // Four 16-key steps of P V: the first or the second half of the tile's keys.
      auto issue_pv = [&](int t, bool second, bool fresh) {
        const uint32_t v = v_low + ((t & 1) ? kTile16 >> 4 : 0) + (second ? 4 * 128 : 0);
        const uint32_t a = s_col + (second ? 32 : 0);
        mma_ts<0>(o_col, a, v, high, !fresh);
        mma_ts<1>(o_col, a, v, high, true);
        mma_ts<2>(o_col, a, v, high, true);
        mma_ts<3>(o_col, a, v, high, true);
      };
      int t = 0, tq = 0, segs = 0;  // key tiles; tiles and segments of this query tile
      bool ok = true;
      for (bool more_segs = w.begin(p, start, n_steps); ok && more_segs; more_segs = w.next(p)) {
        const int count = w.j1 - w.j0;
        if (i == 1 && !w.two(p)) {
          // No rows here: only report the tiles as read once they are there.
          for (int jj = 0; ok && jj < count; ++jj, ++t) {
            if (!(ok = spin_bar(bar(kKFull + (t & 1)), (t >> 1) & 1, abort_flag))) break;
            bar_arrive(bar(kKEmpty + (t & 1)));
            if (!(ok = spin_bar(bar(kVFull + (t & 1)), (t >> 1) & 1, abort_flag))) break;
            bar_arrive(bar(kVEmpty + (t & 1)));
          }
          continue;
        }
        if (!(ok = spin_bar(bar(kQFull + i), segs & 1, abort_flag))) break;
        ++segs;
        // Round jj: P V of tile jj, S of tile jj + 1 (t is tile jj + 1's).
        for (int jj = -1; jj < count; ++jj) {
          const int last = t - 1;  // tile jj's number
          if (jj >= 0) {
            if (!(ok = spin_bar(bar(kVFull + (last & 1)), (last >> 1) & 1, abort_flag))) break;
#pragma unroll 1
            for (int second = 0; second < 2; ++second) {
              if (!(ok = spin_bar(bar((second ? kPFull : kPHalf) + i), tq & 1, abort_flag))) break;
              tc_fence_after();
              issue_pv(last, second, jj == 0 && !second);
            }
            if (!ok) break;
            ++tq;
          }
          if (jj + 1 < count) {
            if (!(ok = spin_bar(bar(kKFull + (t & 1)), (t >> 1) & 1, abort_flag))) break;
            tc_fence_after();
            issue_s(t);
            tc_commit(bar(kSFull + i));
            tc_commit(bar(kKEmpty + (t & 1)));
            ++t;
          } else {
            tc_commit(bar(kOFinal + i));
          }
          if (jj >= 0) tc_commit(bar(kVEmpty + (last & 1)));
        }
      }
      tc_commit(bar(kMmaDone));
    } else if (warp == 15 && lane == 0) {
      // The units that begin here and the CTAs that share each, for the merge.  Nothing is waited for: the merge
      // runs after a CTA that gave up too, and what it takes indices from has to be there all the same.
      for (bool more = w.begin(p, start, n_steps); more; more = w.next(p)) {
        if (w.j0 != 0) continue;
        const int last = static_cast<int>((per * blockIdx.x + w.done + w.steps - 1) / per);
        p.ws_units[w.unit(p)] = make_int4(static_cast<int>(blockIdx.x), last, w.first() ? 0 : 1, 0);
      }
    }
    __syncwarp();
  } else {
    // ------------------------------- softmax -------------------------------
    const int qi = (warp - 4) >> 2;
    const int row = (warp & 3) * 32 + lane;  // row of the query tile = TMEM lane
    const uint32_t lanes = tmem + (static_cast<uint32_t>((warp & 3) * 32) << 16);
    const uint32_t s_addr = lanes + col_s(qi), o_addr = lanes + col_o(qi);
    const int segs_tile = kTileKeys >> shift;
    int n_tiles = 0, n_segs = 0, n_turns = 0;
    const int turn = kTurn + 2 * (warp & 3);  // barrier turn + i: this pair's warp of tile i may go
    bool ok = true;
    for (bool more = w.begin(p, start, n_steps); ok && more; more = w.next(p)) {
      const bool two = w.two(p);
      if (qi == 1 && !two) continue;
      // This thread's query row (rows of the K/V head), its token and its offset in q and out.
      auto q_row = [&] { return w.qb * kUnitRows + qi * kM + row; };
      auto row_at = [&](const int64_t member, const int64_t token_stride) {
        const int r = min(q_row(), p.rows - 1), t = r / p.group;
        return w.b * member + t * token_stride + (w.h * p.group + (r - t * p.group)) * kKv4D;
      };
      const int n = member_len(p, w.b);
      const int lim = token_limit(p, n, min(q_row(), p.rows - 1) / p.group);
      // Rows grow downwards and their limits with them: the first tile in which a row of this query tile
      // does not see every key.
      const int j_mask = token_limit(p, n, min(w.qb * kUnitRows + qi * kM, p.rows - 1) / p.group) / kTileKeys;
      float scale;
      float* const factor = reinterpret_cast<float*>(smem + kOffFactor) + qi * kM + row;
      *factor = 1.f;
      {
        // Q, scaled to fp16 and stored 128-byte swizzled.
        uint4 x[16];
        const __nv_bfloat16* src = p.q + row_at(p.q_member, p.q_row);
        uint32_t top = 0;
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          x[i] = q_row() < p.rows ? *reinterpret_cast<const uint4*>(src + 8 * i) : make_uint4(0, 0, 0, 0);
          top = __vmaxu2(top, __vmaxu2(__vmaxu2(x[i].x & 0x7fff7fffu, x[i].y & 0x7fff7fffu),
                                       __vmaxu2(x[i].z & 0x7fff7fffu, x[i].w & 0x7fff7fffu)));
        }
        float back;
        const float power = row_power(__uint_as_float(max(top << 16, top & 0xffff0000u)), back);
        scale = fmaxf(back * p.scale_log2, 1.2e-38f);  // not 0: a masked score times it stays -inf
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          const uint32_t v[4] = {x[i].x, x[i].y, x[i].z, x[i].w};
          uint32_t o[4];
#pragma unroll
          for (int e = 0; e < 4; ++e)
            o[e] = h2_pack(__uint_as_float(v[e] << 16) * power, __uint_as_float(v[e] & 0xffff0000u) * power);
          const uint32_t dst = sbase + kOffQ + qi * kTile16 + (i >> 3) * kHalf16 + row * 128 + (((i & 7) ^ (row & 7)) * 16);
          asm volatile("st.shared.v4.b32 [%0], {%1,%2,%3,%4};" ::"r"(dst), "r"(o[0]), "r"(o[1]), "r"(o[2]), "r"(o[3])
                       : "memory");
        }
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        tc_fence_before();
        __syncwarp();
        if (lane == 0) bar_arrive(bar(kQFull + qi));
      }
      // Does the segment have a page that is not in the pool?  Its keys are left out, tile by tile.
      auto bad_pages = [&](int first, int end) {  // bit i: page first + 32 k + i, k = 0, 1, .., is not there
        bool bad = false;
        for (int i = first + lane; i < end; i += 32)
          bad |= static_cast<uint32_t>(p.cache.table[w.b * p.cache.table_pages + i]) >= p.cache.num_pages;
        return __ballot_sync(0xffffffffu, bad);
      };
      const int pages_seen = (w.lim_top + (1 << shift) - 1) >> shift;
      // Bit 0: a page that is not there; bit 1: a row of the warp whose scores are scaled in tensor memory.
      int careful = bad_pages(w.j0 * segs_tile, min(w.j1 * segs_tile, pages_seen)) != 0 ? 1 : 0;
      float m = -INFINITY, l = 0.f;
      for (int j = w.j0; j < w.j1; ++j, ++n_tiles) {
        if (!(ok = warp_spin(bar(kSFull + qi), n_tiles & 1, abort_flag))) break;
        tc_fence_after();
        // A tile of which the row does not see every key: -inf over the others, in tensor memory, so that
        // the passes below need not know; nor of scores that are scaled here.
        if (j >= j_mask || careful) {
          if (__builtin_expect(careful & 2, 0)) scale_scores(s_addr, *factor);
          const uint32_t bad = careful & 1 ? bad_pages(j * segs_tile, min((j + 1) * segs_tile, pages_seen)) : 0;
          const int valid = lim - j * kTileKeys;
#pragma unroll 1
          for (int col = 0; col < 128; col += 16) {
            uint32_t y[16];
            tmem_ld16(s_addr + col, y);
            tmem_wait_ld16(y);
#pragma unroll
            for (int i = 0; i < 16; ++i)
              if (col + i >= valid || ((bad >> ((col + i) >> shift)) & 1)) y[i] = __float_as_uint(-INFINITY);
            tmem_st16(s_addr + col, y);
          }
          tmem_wait_st();
        }
        // Two passes over the scores in tensor memory, 32 columns at a time with the next 32 on their way:
        // the row's maximum, then the probabilities.  The loops stay rolled: a sub-partition runs
        // four roles' code side by side, and unrolled they wait for instructions more than for anything
        // else (the 1.3B block call took 600 us with this loop unrolled).
        uint32_t xa[32], xb[32];
        float mx[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
        auto largest = [&](const uint32_t* y) {
#pragma unroll
          for (int i = 0; i < 32; i += 2)
            mx[(i >> 1) & 3] = max3(mx[(i >> 1) & 3], __uint_as_float(y[i]), __uint_as_float(y[i + 1]));
        };
        tmem_ld32(s_addr, xa);
#pragma unroll 1
        for (int col = 0; col < 128; col += 64) {
          tmem_wait_ld32(xa);
          tmem_ld32(s_addr + col + 32, xb);
          largest(xa);
          tmem_wait_ld32(xb);
          tmem_ld32(s_addr + ((col + 64) & 127), xa);  // the last one is the second pass's first
          largest(xb);
        }
        const float top = fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3])) * scale;
        const bool grow = top > most_of(m);
        const float next = grow ? reference_of(top) : m;
        const float alpha = grow ? fast_exp2(m - next) : 1.f;
        if (grow) {
          l *= alpha;
          m = next;
        }
        if (__any_sync(0xffffffffu, grow)) {
          // O holds this segment's earlier tiles (their P V have completed: S was committed after them).
          if (j > w.j0) {
#pragma unroll 1
            for (int c = 0; c < 8; ++c) {
              uint32_t o[16];
              tmem_ld16(o_addr + 16 * c, o);
              tmem_wait_ld16(o);
#pragma unroll
              for (int i = 0; i < 16; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * alpha);
              tmem_st16(o_addr + 16 * c, o);
            }
          }
          const bool far = grow && !(fabsf(m) < kNear) && scale != 1.f;  // (once: its scale is 1 then)
          if (__builtin_expect(__any_sync(0xffffffffu, far), 0)) {
            careful |= 2;
            tmem_wait_ld32(xa);
            scale_scores(s_addr, far ? scale : 1.f);
            tmem_ld32(s_addr, xa);
            if (far) {
              *factor = scale;
              scale = 1.f;
            }
          }
        }
        const float ref = m == -INFINITY ? 0.f : m;
        const f32x2 scale2 = f2_make(scale, scale), ref2 = f2_make(-ref, -ref);
        f32x2 sum[2] = {0, 0};
        // Tile 0's k-th turn follows tile 1's (k-1)-th, tile 1's k-th follows tile 0's k-th.
        if (two) {
          if (qi + n_turns > 0 && !(ok = warp_spin(bar(turn + qi), (n_turns - 1 + qi) & 1, abort_flag))) break;
          ++n_turns;
        }
        // 32 scores to probabilities, over columns that both passes have read.
        auto exponentiate = [&](const uint32_t* y, uint32_t p_col) {
          uint32_t pk[16];
#pragma unroll
          for (int c = 0; c < 16; ++c) {
            float x0, x1;
            f2_split(f2_fma(f2_make(__uint_as_float(y[2 * c]), __uint_as_float(y[2 * c + 1])), scale2, ref2), x0, x1);
            x0 = fast_exp2(x0);
            x1 = fast_exp2(x1);
            sum[c & 1] = f2_add(sum[c & 1], f2_make(x0, x1));
            pk[c] = h2_pack(x0, x1);
          }
          tmem_st16(s_addr + p_col, pk);
        };
#pragma unroll 1
        for (int col = 0; col < 128; col += 64) {
          tmem_wait_ld32(xa);
          tmem_ld32(s_addr + col + 32, xb);
          exponentiate(xa, col >> 1);
          tmem_wait_ld32(xb);
          if (col == 0) tmem_ld32(s_addr + 64, xa);
          exponentiate(xb, (col >> 1) + 16);
          if (col != 0 && two && lane == 0) bar_arrive(bar(turn + 1 - qi));
          tmem_wait_st();
          tc_fence_before();
          __syncwarp();
          if (lane == 0) bar_arrive(bar((col == 0 ? kPHalf : kPFull) + qi));
        }
        float l0, l1;
        f2_split(f2_add(sum[0], sum[1]), l0, l1);
        l += l0 + l1;
      }
      if (!ok) break;
      if (!(ok = warp_spin(bar(kOFinal + qi), n_segs & 1, abort_flag))) break;
      ++n_segs;
      tc_fence_after();
      const bool live = q_row() < p.rows;
      if (w.whole()) {
        const float inv = l == 0.f ? 0.f : p.cache.v_scale / l;
        __nv_bfloat16* dst = p.out + row_at(p.out_member, p.out_row);
#pragma unroll 1
        for (int c = 0; c < 4; ++c) {
          uint32_t o[32];
          tmem_ld32(o_addr + 32 * c, o);
          tmem_wait_ld32(o);
          if (live) {
#pragma unroll
            for (int v = 0; v < 4; ++v) {
              uint32_t y[4];
#pragma unroll
              for (int e = 0; e < 4; ++e)
                y[e] = l == 0.f ? 0u
                                : Pairs16<__nv_bfloat16>::pack_pair(__uint_as_float(o[8 * v + 2 * e]) * inv,
                                                                    __uint_as_float(o[8 * v + 2 * e + 1]) * inv);
              *reinterpret_cast<uint4*>(dst + 32 * c + 8 * v) = make_uint4(y[0], y[1], y[2], y[3]);
            }
          }
        }
      } else {
        const int64_t slot = (2ll * blockIdx.x + (w.first() ? 0 : 1)) * kUnitRows + qi * kM + row;
        float* dst = p.ws_o + slot * kKv4D;
#pragma unroll 1
        for (int c = 0; c < 4; ++c) {
          uint32_t o[32];
          tmem_ld32(o_addr + 32 * c, o);
          tmem_wait_ld32(o);
#pragma unroll
          for (int v = 0; v < 4; ++v)
            asm volatile("st.global.v8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"l"(dst + 32 * c + 8 * v), "r"(o[8 * v]),
                         "r"(o[8 * v + 1]), "r"(o[8 * v + 2]), "r"(o[8 * v + 3]), "r"(o[8 * v + 4]), "r"(o[8 * v + 5]),
                         "r"(o[8 * v + 6]), "r"(o[8 * v + 7])
                         : "memory");
        }
        p.ws_ml[slot] = make_float2(m, l);
      }
      tc_fence_before();
    }
  }

  // Teardown: every role has left its loop; wait for the MMAs in flight, free the tensor memory.
  pdl_trigger();
  __syncthreads();
  if (warp == 12) {
    if (lane == 0) {
      volatile int never = 0;
      spin_bar(bar(kMmaDone), 0, &never);
    }
    __syncwarp();
    tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512) : "memory");
  }
}

// Merges the segments of the units that several CTAs of the tiles kernel shared.  A warp per query row.
__global__ void __launch_bounds__(256) kv4_merge_kernel(const __grid_constant__ AParams p) {
  pdl_wait();
  const int lane = threadIdx.x & 31;
  const int64_t unit = blockIdx.x / (kUnitRows / 8);
  const int r = static_cast<int>(blockIdx.x % (kUnitRows / 8)) * 8 + (threadIdx.x >> 5);
  const int4 info = p.ws_units[unit];  // first CTA, last CTA, slot of the first CTA
  if (info.x == info.y) return;
  const int64_t bh = unit / p.row_blocks;
  const int row = static_cast<int>(unit - bh * p.row_blocks) * kUnitRows + r;
  if (row >= p.rows) return;
  auto slot_of = [&](int cta) { return (2ll * cta + (cta == info.x ? info.z : 0)) * kUnitRows + r; };
  float top = -INFINITY, sum = 0.f;
  for (int c = info.x; c <= info.y; ++c) top = fmaxf(top, p.ws_ml[slot_of(c)].x);
  float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
  for (int c = info.x; c <= info.y; ++c) {
    const int64_t slot = slot_of(c);
    const float2 ml = p.ws_ml[slot];
    if (ml.y == 0.f) continue;  // the row saw nothing there
    const float f = ml.x == top ? 1.f : fast_exp2(ml.x - top);
    const float4 y = *reinterpret_cast<const float4*>(p.ws_o + slot * kKv4D + 4 * lane);
    sum += f * ml.y;
    x.x += f * y.x;
    x.y += f * y.y;
    x.z += f * y.z;
    x.w += f * y.w;
  }
  const float inv = sum == 0.f ? 0.f : p.cache.v_scale / sum;
  const int b = static_cast<int>(bh / p.cache.kv_heads), h = static_cast<int>(bh % p.cache.kv_heads), t = row / p.group;
  __nv_bfloat16* dst = p.out + b * p.out_member + t * p.out_row + (h * p.group + (row - t * p.group)) * kKv4D + 4 * lane;
  *reinterpret_cast<uint2*>(dst) = make_uint2(Pairs16<__nv_bfloat16>::pack_pair(x.x * inv, x.y * inv),
                                              Pairs16<__nv_bfloat16>::pack_pair(x.z * inv, x.w * inv));
}

// ---------------------------------------------------------------------------------------
// Host side
// ---------------------------------------------------------------------------------------
struct APlan {
  AParams params;
  int kernel;       // ps_kv4_kernel, resolved
  int64_t ctas;     // rows kernel: grid
  int64_t ws_bytes;
};

// Key chunks per unit: the least modelled time, in tile times of one CTA.  `slots` CTAs run at once; a
// CTA takes about three tile times to start and finish; partial results cost a second launch.
static int choose_chunks(int64_t units, int tiles, int64_t slots) {
  int best = 1;
  double best_cost = 0;
  for (int c = 1; c <= kMaxChunks && c <= tiles; ++c) {
    const int64_t waves = (units * c + slots - 1) / slots;
    const double cost = static_cast<double>(waves) * ((tiles + c - 1) / c + 3) + (c > 1 ? 4 : 0);
    if (c == 1 || cost < best_cost) {
      best = c;
      best_cost = cost;
    }
  }
  return best;
}

static int check_rows(const void* ptr, int64_t member, int64_t row, int64_t C, int64_t members, int64_t rows,
                      const char* name) {
  if (!ptr) return fail(PS_ERR_NULL, "%s is NULL", name);
  if (!aligned16(ptr)) return fail(PS_ERR_ALIGN, "%s is not 16-byte aligned", name);
  if (row < C) return fail(PS_ERR_SHAPE, "%s row stride %lld is below its %lld columns", name, (long long)row, (long long)C);
  if ((row * 2) % 16 || (members > 1 && (member * 2) % 16))
    return fail(PS_ERR_ALIGN, "%s strides must be multiples of 16 bytes", name);
  if (members > 1 && member < rows * row)
    return fail(PS_ERR_SHAPE, "%s member stride %lld overlaps %lld rows", name, (long long)member, (long long)rows);
  return PS_OK;
}

static int build_attn(const ps_kv4_attn_args* a, APlan* plan, bool host_only) {
  clear_error();
  if (!a) return fail(PS_ERR_NULL, "args is NULL");
  memset(plan, 0, sizeof(*plan));
  AParams& p = plan->params;
  int64_t cache_rows = 0;
  int rc = kv4_check_cache(a->cache, &p.cache, &cache_rows);
  if (rc) return rc;
  const int hk = a->cache.kv_heads;
  if (a->heads < 1 || a->heads % hk)
    return fail(PS_ERR_SHAPE, "heads=%d is not a multiple of kv_heads=%d", a->heads, hk);
  // The kernels take the columns of a token in 32 bits.
  if (a->heads > INT32_MAX / kKv4D) return fail(PS_ERR_UNSUPPORTED, "heads=%d: columns beyond 2^31", a->heads);
  if (a->q_tokens < 0 || a->kv_tokens < 0 || a->causal_block < 0)
    return fail(PS_ERR_SHAPE, "q_tokens=%d kv_tokens=%d causal_block=%d", a->q_tokens, a->kv_tokens, a->causal_block);
  if (a->kv_tokens > a->cache.table_pages * a->cache.page_rows)
    return fail(PS_ERR_BOUNDS, "kv_tokens=%d exceeds a member's %lld cache rows", a->kv_tokens,
                (long long)(a->cache.table_pages * a->cache.page_rows));
  if (a->kv_tokens > (1 << 30)) return fail(PS_ERR_UNSUPPORTED, "kv_tokens=%d beyond 2^30", a->kv_tokens);
  if (a->kernel != PS_KV4_AUTO && a->kernel != PS_KV4_ROWS && a->kernel != PS_KV4_TILES)
    return fail(PS_ERR_SHAPE, "kernel %d unknown", a->kernel);
  if (a->key_chunks < 0 || a->key_chunks > kMaxChunks)
    return fail(PS_ERR_SHAPE, "key_chunks=%d (0..%d)", a->key_chunks, kMaxChunks);
  const int64_t C = static_cast<int64_t>(a->heads) * kKv4D;
  if ((rc = check_rows(a->q, a->q_member_stride, a->q_row_stride, C, a->cache.members, a->q_tokens, "q")) ||
      (rc = check_rows(a->out, a->out_member_stride, a->out_row_stride, C, a->cache.members, a->q_tokens, "out")))
    return rc;
  if (reinterpret_cast<uintptr_t>(a->kv_lens) & 3u) return fail(PS_ERR_ALIGN, "kv_lens is not 4-byte aligned");
  p.q = static_cast<const __nv_bfloat16*>(a->q);
  p.out = static_cast<__nv_bfloat16*>(a->out);
  p.lens = a->kv_lens;
  p.q_member = a->q_member_stride; p.q_row = a->q_row_stride;
  p.out_member = a->out_member_stride; p.out_row = a->out_row_stride;
  p.Lq = a->q_tokens;
  p.kv_max = a->kv_tokens;
  p.causal_block = a->causal_block;
  p.group = a->heads / hk;
  const int64_t rows = static_cast<int64_t>(a->q_tokens) * p.group;
  if (rows > (1 << 30)) return fail(PS_ERR_UNSUPPORTED, "%lld query rows of a K/V head", (long long)rows);
  p.rows = static_cast<int32_t>(rows);
  const int tiles = (a->kv_tokens + kTileKeys - 1) / kTileKeys;
  const int sms = sm_count();
  plan->kernel = a->kernel;
  if (plan->kernel == PS_KV4_AUTO) {
    // The rows kernel passes over the keys once per 8 query rows, 0.62 us a 128-key tile on an SM; the tiles
    // kernel once per 256 rows, about 2.2 us, and it takes 13 us to start and finish against 6 (measured).
    // Per K/V head they meet between 24 and 32 rows on long windows (12 heads over 34 320 keys: 24 rows 48
    // us against 68, 32 rows 60 against 68, 64 rows 112 against 70) and past 128 on short ones (1 024 keys:
    // 15 us against 16).
    const double heads_tiles = static_cast<double>(a->cache.members) * hk * tiles / sms;
    const double rows_us = 6 + 0.62 * heads_tiles * ((rows + kBlockRows - 1) / kBlockRows);
    const double tiles_us = 13 + 2.2 * heads_tiles * ((rows + kUnitRows - 1) / kUnitRows);
    plan->kernel = rows_us <= tiles_us ? PS_KV4_ROWS : PS_KV4_TILES;
  }
  const bool tiles_kernel = plan->kernel == PS_KV4_TILES;
  const int block_rows = tiles_kernel ? kUnitRows : kBlockRows;
  p.row_blocks = (p.rows + block_rows - 1) / block_rows;
  if (p.row_blocks > 0 && a->cache.members * hk > (1 << 25) / p.row_blocks)
    return fail(PS_ERR_UNSUPPORTED, "%lld members of %d K/V heads and %d row blocks", (long long)a->cache.members, hk,
                p.row_blocks);
  p.units = a->cache.members * hk * p.row_blocks;
  const double scale = a->scale > 0.f ? a->scale : 1.0 / sqrt(static_cast<double>(kKv4D));
  p.scale_log2 = static_cast<float>(scale * a->cache.k_scale * 1.4426950408889634);
  int64_t slots;
  if (tiles_kernel) {
    p.chunks = 1;
    p.min_steps = 2;
    p.grid = sms;
    // With fixed lengths the number of steps is known: no CTA without work.
    const int64_t most = p.units * (tiles > 0 ? tiles : 1);
    if ((most + p.min_steps - 1) / p.min_steps < p.grid) p.grid = static_cast<int32_t>((most + p.min_steps - 1) / p.min_steps);
    slots = 2ll * p.grid * kUnitRows;
    // The partial rows go out 32 bytes at a time: they start at the workspace's first 32-byte boundary.
    plan->ws_bytes = slots * (kKv4D * 4 + 8) + p.units * static_cast<int64_t>(sizeof(int4)) + 16;
  } else {
    int chunks = a->key_chunks > 0 ? a->key_chunks : choose_chunks(p.units, tiles, 3ll * sms);
    if (chunks > tiles) chunks = tiles > 0 ? tiles : 1;
    p.chunks = chunks;
    plan->ctas = p.units * chunks;
    if (a->kv_lens && a->key_chunks == 0 && chunks > 1 && p.units <= sms) {
      // Few units of work of lengths that the host does not know: the device splits them by length.  One wave
      // of CTAs, or up to four while a chunk keeps a dozen tiles (of windows half as long as they may be).
      // 7 members x 12 rows of 8 K/V heads over 1 024 .. 8 191 keys (112 units): 26 us, equal chunks 30.  With
      // more units than SMs the waves even the lengths out by themselves, and the split only costs its
      // planning (200 units of 375 .. 3 000 keys: 27.3 us, equal chunks 26.4).
      const int64_t wave = 3ll * sms, waves = p.units * tiles / (2 * wave * 12);
      p.chunks = 0;
      plan->ctas = wave * (waves < 1 ? 1 : waves > 4 ? 4 : waves);
    }
    slots = plan->ctas * kBlockRows;
    plan->ws_bytes = chunks > 1 ? slots * (kKv4D * 4 + 8) : 0;
    if (p.chunks == 0) plan->ws_bytes += a->cache.members * static_cast<int64_t>(sizeof(int4));
  }
  if (plan->ctas > 0x7fffffffLL) return fail(PS_ERR_UNSUPPORTED, "grid of %lld CTAs", (long long)plan->ctas);
  if (!host_only && plan->ws_bytes > 0) {
    if (!a->workspace || a->workspace_bytes < plan->ws_bytes)
      return fail(PS_ERR_NULL, "workspace of %lld bytes needed (ps_kv4_attention_workspace), %lld given",
                  (long long)plan->ws_bytes, (long long)a->workspace_bytes);
    if (!aligned16(a->workspace)) return fail(PS_ERR_ALIGN, "workspace is not 16-byte aligned");
  }
  unsigned char* base = static_cast<unsigned char*>(a->workspace);
  if (tiles_kernel && (reinterpret_cast<uintptr_t>(base) & 31u)) base += 16;
  p.ws_o = reinterpret_cast<float*>(base);
  p.ws_ml = reinterpret_cast<float2*>(base + slots * kKv4D * 4);
  p.ws_units = reinterpret_cast<int4*>(p.ws_ml + slots);
  return PS_OK;
}

// Opts `fn` into `bytes` of dynamic shared memory, once per device.
static cudaError_t allow_smem(const void* fn, int bytes) {
  static const void* done[64][4];
  static std::mutex lock;
  int dev = 0;
  cudaError_t err = cudaGetDevice(&dev);
  if (err != cudaSuccess) return err;
  std::lock_guard<std::mutex> guard(lock);
  if (dev >= 0 && dev < 64)
    for (const void*& f : done[dev]) {
      if (f == fn) return cudaSuccess;
      if (!f) {
        err = cudaFuncSetAttribute(fn, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
        if (err == cudaSuccess) f = fn;
        return err;
      }
    }
  return cudaFuncSetAttribute(fn, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
}

template <typename... A>
static cudaError_t launch(void (*fn)(A...), int64_t blocks, int threads, int smem, cudaStream_t stream,
                          std::common_type_t<A>... args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(blocks));
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, fn, args...);
}

}  // namespace

cudaError_t kv4_attention_counts(uint32_t* counts, int reset) { return kv4_take_counts(counts, reset); }

}  // namespace ps

extern "C" int32_t ps_kv4_attention_validate(const ps_kv4_attn_args* args) {
  ps::APlan plan;
  return ps::build_attn(args, &plan, true);
}

extern "C" int32_t ps_kv4_attention_workspace(const ps_kv4_attn_args* args, int64_t* bytes) {
  if (!bytes) return ps::fail(PS_ERR_NULL, "bytes is NULL");
  ps::APlan plan;
  const int rc = ps::build_attn(args, &plan, true);
  if (rc == PS_OK) *bytes = plan.ws_bytes;
  return rc;
}

extern "C" int32_t ps_attention_kv4(const ps_kv4_attn_args* args, void* stream) {
  ps::APlan plan;
  const int rc = ps::build_attn(args, &plan, false);
  if (rc != PS_OK || plan.params.units == 0) return rc;
  const ps::AParams& p = plan.params;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (plan.kernel == PS_KV4_TILES) {
    cudaError_t err = ps::allow_smem(reinterpret_cast<const void*>(ps::kv4_tiles_kernel), ps::kTilesSmem);
    if (err == cudaSuccess)
      err = ps::launch(ps::kv4_tiles_kernel, p.grid, ps::kTilesThreads, ps::kTilesSmem, s, p, args->cache.members);
    if (err == cudaSuccess)
      err = ps::launch(ps::kv4_merge_kernel, p.units * (ps::kUnitRows / 8), 256, 0, s, p);
    if (err != cudaSuccess) return ps::fail(PS_ERR_LAUNCH, "kv4 attention launch: %s", cudaGetErrorString(err));
    return PS_OK;
  }
  const int smem = static_cast<int>(sizeof(ps::RowsShared)) + 128;
  cudaError_t err = ps::allow_smem(reinterpret_cast<const void*>(ps::kv4_rows_kernel), smem);
  if (err == cudaSuccess) err = ps::launch(ps::kv4_rows_kernel, plan.ctas, ps::kRowThreads, smem, s, p);
  if (err == cudaSuccess && p.chunks != 1) {
    const int64_t rows = p.units / p.row_blocks * p.rows;
    err = ps::launch(ps::kv4_combine_kernel, (rows + 3) / 4, 128, 0, s, p);
  }
  if (err != cudaSuccess) return ps::fail(PS_ERR_LAUNCH, "kv4 attention launch: %s", cudaGetErrorString(err));
  return PS_OK;
}
