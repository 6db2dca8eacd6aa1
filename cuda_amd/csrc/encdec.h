// What the attention of encoder-decoder models has beside q, k and v of one
// length: keys of another length, padded per sequence (cross attention), and a
// learned relative position bias by buckets.
//
// Kernels take one of three types X: SelfX (one length, nothing else), CrossX
// (a key length per sequence) or BiasX (CrossX and a bias per distance).
//
// The bias of query i and key j of head h is table[bucket(j - i)][h]. Buckets
// are given by the first distance of each of a side's: bucket(n) is the last b
// with first[b] <= n, n = |j - i|; keys after their query (j > i) have a side of
// their own unless only those before it count (one_sided: n = 0 there). Past
// `reach`, the last bucket's first distance, the bias of a side is one value.
// Kernels keep a head's bias by distance in LDS, [-(reach + 96), reach + 95] (one
// side: up to 95), and move a block whose distances all lie past the reach into
// that margin.
#pragma once

#include <algorithm>

#include "common.h"
#include "launch.h"
#include "lds_dma.h"

namespace ca {

constexpr int kMaxBuckets = 256;   // of both sides; an id fits a byte
constexpr int kMaxReach = 2048;    // 17 KB of bias by distance beside the rings
constexpr int kBiasMargin = 96;    // a block's distances span at most 95

// A finite bias is brought into [-2^15, 2^15]: one that low already takes all
// weight from a key beside any other, and float32 logits of that size keep
// their differences to 2^-8. -inf stays (the key takes no part).
constexpr float kMaxBias = 32768.f;

struct SelfX {
  static constexpr bool kCross = false, kBias = false;
  struct Grad {};
};

struct CrossX {
  static constexpr bool kCross = true, kBias = false;
  struct Grad {};
  const int32_t* kv_lens;  // [B], null: Skv for all
  int Skv, B;
  // Head j of a launch's order among `per_b` heads of each sequence. A sequence's
  // heads lie apart, so that every XCD's share of the order (an eighth, common.h)
  // has all sequences in it, whatever their lengths; where 8 divides per_b, an XCD
  // takes its heads of the longest sequence first, and the short ones fill the end.
  // (4 x 32 heads x 2048 queries, 1792 to 4096 keys: 466 us head by head, when two
  // XCDs had the longest sequence to themselves; 383 apart; 360 longest first.)
  struct Head {
    int bh, n_keys;  // the head, its sequence's keys
  };
  __device__ __forceinline__ Head head(int j, int per_b) const {
    auto plain = [&](int b, int h) CA_INLINE {
      const int n = kv_lens ? kv_lens[b] : Skv;
      return Head{b * per_b + h, __builtin_amdgcn_readfirstlane(min(max(n, 0), Skv))};
    };
    if (per_b % 8) return plain(j % B, j / B);
    const int hx = per_b / 8, share = hx * B, xcd = j / share, i = j % share;
    const int r = i / hx, h = xcd * hx + i % hx;
    if (!kv_lens || B == 1 || B > 64) return plain(r, h);
    // the sequence of rank r by length: lane l counts those that come before l
    const int lane = lane_here();
    const int n = lane < B ? min(max(kv_lens[lane], 0), Skv) : -1;
    int rank = 0;
    for (int l = 0; l < B; ++l) {
      const int m = __builtin_amdgcn_readlane(n, l);
      rank += m > n || (m == n && l < lane);
    }
    const int b = __builtin_ctzll(__ballot(lane < B && rank == r));
    return Head{b * per_b + h, __builtin_amdgcn_readlane(n, b)};
  }
  // keys of sequence b
  __device__ __forceinline__ int kv_len(int b) const {
    const int n = kv_lens ? kv_lens[b] : Skv;
    return __builtin_amdgcn_readfirstlane(min(max(n, 0), Skv));
  }
};

struct BiasGrad;
struct BiasGradWide;
struct BiasX : CrossX {
  static constexpr bool kBias = true, kWide = false;
  using Grad = BiasGrad;
  const void* table;   // [buckets][Hq] of table_dtype
  int table_dtype;     // kDtypeF32, ...
  float mul;           // table values times this are the kernel's
  float scale_log2;    // ... which, times this, are log2 logits
  int side;            // buckets of a side
  int one_sided;       // keys after their query: distance 0
  int reach;           // distances from here on are in a side's last bucket
  int Hq;
  uint16_t first[kMaxBuckets];  // first distance of a side's bucket
  __host__ __device__ __forceinline__ int buckets() const { return one_sided ? side : 2 * side; }
  __device__ __forceinline__ float value(int bucket, int h) const;
};

// BiasX of a dQ launch whose LDS does not hold BiasGrad
struct BiasWideX : BiasX {
  static constexpr bool kWide = true;
  using Grad = BiasGradWide;
};

// ---------------------------------------------------------------------------
// A head's bias by distance in LDS (dynamic: bias_lds_bytes)
// ---------------------------------------------------------------------------
__host__ __device__ __forceinline__ int bias_entries(const BiasX& x) {
  return x.reach + (x.one_sided ? 0 : x.reach) + 2 * kBiasMargin;
}
__host__ __device__ __forceinline__ size_t bias_lds_bytes(const BiasX& x) { return 4 * (size_t)bias_entries(x); }

__device__ __forceinline__ float bias_clamp(float v) {
  // (not by min and max: a NaN and -inf stay)
  v = v > kMaxBias && v != -kNegInf ? kMaxBias : v;
  return v < -kMaxBias && v != kNegInf ? -kMaxBias : v;
}

// The kernel's bias of a bucket: clamped, times mul.
__device__ __forceinline__ float BiasX::value(int bucket, int h) const {
  const size_t i = (size_t)bucket * Hq + h;
  float v;
  if (table_dtype == kDtypeF32) v = ((const float*)table)[i];
  else if (table_dtype == kDtypeBF16) v = BF16::to_float(((const uint16_t*)table)[i]);
  else v = F16::to_float(((const uint16_t*)table)[i]);
  return bias_clamp(v) * mul;
}

// The entries of a bucket's distances: from n0 to before n1, distance n of those
// at or before their query at zero - n, of the others (from 1 on) at zero + n.
// The last bucket of a side has the margin.
struct BucketRange {
  int n0, n1, sign;
};
__device__ __forceinline__ BucketRange bucket_range(const BiasX& x, int b) {
  const bool after = b >= x.side;
  const int s = after ? b - x.side : b;
  const int end = x.reach + kBiasMargin + (after ? 0 : 1);
  return {max((int)x.first[s], after ? 1 : 0), s + 1 < x.side ? min((int)x.first[s + 1], end) : end, after ? 1 : -1};
}

// write(entry, value(bucket)) for all entries, 16 threads to a bucket: a value is
// one load, and its entries a few writes behind it (searching each entry's bucket
// took 1.2 us a workgroup).
template <class V, class W>
__device__ __forceinline__ void bias_spread(const BiasX& x, int threads, V value, W write) {
  // (not from the work-item id, which would stay in a register up to here)
  const int tid = 64 * __builtin_amdgcn_readfirstlane(threadIdx.x >> 6) + lane_here();
  const int zero = x.reach + kBiasMargin, buckets = x.buckets();
  for (int b = tid >> 4; b < buckets; b += threads >> 4) {
    const auto v = value(b);
    const BucketRange r = bucket_range(x, b);
    for (int n = r.n0 + (tid & 15); n < r.n1; n += 16) write(zero + r.sign * n, v);
  }
}

// Fills the workgroup's bias of head h at `mem` (all threads; ends with a
// barrier). Returns the LDS byte offset of distance 0's entry. DMA: tile loads are
// in flight, which the compiler would wait for before LDS writes of its own; then
// LDS reads are hand-issued too.
template <bool DMA>
__device__ __forceinline__ uint32_t bias_fill(const BiasX& x, int h, unsigned char* mem, int threads) {
  float* e = (float*)mem;
  const uint32_t base = lds_off(mem);
  auto write = [&](int i, float v) CA_INLINE {
    if constexpr (DMA) lds_write_b32<0>(base + 4 * i, v);
    else e[i] = v;
  };
  bias_spread(x, threads, [&](int b) CA_INLINE { return x.value(b, h); }, write);
  if (x.one_sided) {  // (masked: any finite number)
    const int tid = 64 * __builtin_amdgcn_readfirstlane(threadIdx.x >> 6) + lane_here();
    for (int n = 1 + tid; n < kBiasMargin; n += threads) write(x.reach + kBiasMargin + n, 0.f);
  }
  if constexpr (DMA) {
    wait_lgkm<0>();
    __builtin_amdgcn_s_barrier();
  } else {
    __syncthreads();
  }
  return base + 4 * (x.reach + kBiasMargin);
}

// Distance 0's entry in what bias_fill<false> has filled.
__device__ __forceinline__ const float* bias_zero(const BiasX& x, const unsigned char* mem) {
  return (const float*)mem + x.reach + kBiasMargin;
}

// Whether a block of distances [r0, r0 + SPAN] meets more than a side's last
// bucket, and that bucket's bias if not: before their queries, or after.
template <int SPAN>
__device__ __forceinline__ bool bias_near(const BiasX& x, int r0) {
  return r0 <= x.reach && r0 + SPAN >= -x.reach;
}
struct FarBias {
  float before, after;
  __device__ __forceinline__ float of(int r0) const { return r0 > 0 ? after : before; }
};
__device__ __forceinline__ FarBias far_bias(const BiasX& x, uint32_t zero) {
  uint32_t a = lds_read_b32<0>(zero - 4 * (x.reach + kBiasMargin));
  uint32_t b = lds_read_b32<0>(zero + 4 * (bias_entries(x) - x.reach - kBiasMargin - 1));
  wait_lgkm<0>();
  after_wait(a);
  after_wait(b);
  return {__builtin_bit_cast(float, __builtin_amdgcn_readfirstlane(a)),
          __builtin_bit_cast(float, __builtin_amdgcn_readfirstlane(b))};
}

// First distance of a block of distances [r0, r0 + 94], moved into the margin
// where all of them lie past the reach.
__device__ __forceinline__ int bias_block(const BiasX& x, int r0) {
  return min(max(r0, -(x.reach + kBiasMargin - 1)), x.one_sided ? 1 : x.reach + 1);
}

// LDS dwords at a + 4 O0 and a + 4 O1
template <int O0, int O1>
__device__ __forceinline__ u32x2 lds_read2_b32(uint32_t a) {
  u32x2 r = {a, a};
  CA_DEVICE_ASM("ds_read2_b32 %0, %1 offset0:%2 offset1:%3" : "=v"(r) : "v"(a), "n"(O0), "n"(O1));
  return r;
}

// ---------------------------------------------------------------------------
// One query at the end of its keys (decode): distances 0, -1, ...
// ---------------------------------------------------------------------------
// In LDS the bucket ids of distances 0 .. reach (n before the query) and the
// table's columns of up to 16 heads, [bucket][16], in log2 units: a token's
// bias is two reads for each head, and past the reach one value.
struct DecodeBias {
  uint32_t ids, column;  // LDS byte offsets; column: the lane's head
  int reach;
  float far;             // the lane's head from `reach` on
};
constexpr size_t decode_bias_lds_bytes(int side, int reach) {
  return 64 * (size_t)side + (size_t)(reach + 16) / 16 * 16;
}
// All threads; ends with a barrier. Heads h0 .. h0 + n_heads - 1; the lane's is l16.
__device__ __forceinline__ DecodeBias decode_bias_fill(const BiasX& x, int h0, int n_heads, unsigned char* mem,
                                                       int threads, int l16) {
  float* col = (float*)mem;
  unsigned char* ids = (unsigned char*)(col + 16 * x.side);
  for (int i = threadIdx.x; i < 16 * x.side; i += threads)
    col[i] = (i & 15) < n_heads ? x.value(i >> 4, h0 + (i & 15)) : 0.f;
  bias_spread(x, threads, [](int b) CA_INLINE { return b; }, [&](int e, int b) CA_INLINE {
    const int n = x.reach + kBiasMargin - e;
    if (n <= x.reach) ids[n] = (unsigned char)b;
  });
  __syncthreads();
  return {lds_off(ids), lds_off(col + l16), x.reach, col[16 * ids[x.reach] + l16]};
}
// bias of the 8 tokens n0 - i (i = 0 .. 3) and n0 - 16 - i before the query (one
// before it, of a masked token, counts as 0)
__device__ __forceinline__ void decode_bias(const DecodeBias& d, int n0, float (&e)[8]) {
  uint32_t id[8], v[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) id[i] = lds_read_u8<0>(d.ids + min(max(n0 - 16 * (i >> 2) - (i & 3), 0), d.reach));
  wait_lgkm<0>();
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    after_wait(id[i]);
    v[i] = lds_read_b32<0>(d.column + 64 * id[i]);
  }
  wait_lgkm<0>();
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    after_wait(v[i]);
    e[i] = __builtin_bit_cast(float, v[i]);
  }
}

// ---------------------------------------------------------------------------
// The table's gradient: sums of dS by bucket
// ---------------------------------------------------------------------------
// A wave has 32 x 32 blocks of dS (lane l32: query, 16 registers: keys; HALF = 8:
// register r of half hl is key 8 hl + 16 (r / 8) + r % 8, HALF = 16: key 16 hl + r)
// whose 63 distances start at r0. Blocks that lie wholly past the reach on one
// side are one bucket: each lane adds its registers to a running sum of the side.
// No sum depends on timing: each has one writer at a time, in program order. LDS
// accesses are hand-issued: the compiler would wait for the tile loads in flight
// before its own.
//
// BiasGrad (HALF = 8): in LDS a sum for every distance (bias_entries), for each
// wave and lane half. Within a row of 16 lanes (queries j) and a run of 8 keys e,
// shifting by a lane between two keys adds up distances: y = ds[e] + (y of lane j
// + 1), e falling, leaves distance -j in lane j (all of it), and z = ds[e] + (z of
// lane j - 1), e rising, distance 7 - j, of which 7 .. 1 (lanes 0 .. 6) are z's
// alone. The row's z belongs 9 lanes up beside the y of the row 16 distances
// ahead; the four rows and two runs then meet in two registers, whose 64 lanes
// each have a distance of their own half, read, added to and written back. (LDS
// float atomics take a cycle a lane: 16 x 64 of them made a block three times as
// long; through LDS with a segmented scan it took 1.5 us.)
template <int CTRL>
__device__ __forceinline__ float dpp(float x) {
  return __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, x), CTRL, 0xf, 0xf, true));
}
struct BiasGrad {
  static constexpr bool kByDistance = true;  // finish's sums are by distance
  uint32_t at_m, at_q;  // LDS: the lane's entries of the two registers, of a block from distance 0
  float run[2];         // the lane's sums of the blocks past the reach, before and after
  float* mem;           // [waves][2][bias_entries]

  static size_t lds_bytes(const BiasX& x, int waves) { return (size_t)waves * 2 * bias_entries(x) * sizeof(float); }

  // (all threads; a barrier must follow)
  template <int HALF>
  __device__ __forceinline__ void init(const BiasX& x, float* m, int /*buckets*/, int wave, int waves) {
    static_assert(HALF == 8, "runs of 8 keys, the halves' 8 apart");
    const int lane = lane_here(), j = lane & 15, qh = (lane >> 4) & 1, hl = lane >> 5, n = bias_entries(x);
    mem = m;
    run[0] = run[1] = 0.f;
    for (int i = 64 * wave + lane; i < waves * 2 * n; i += 64 * waves) m[i] = 0.f;
    // (r0 is 31 before the distance of the block's first key and query)
    const uint32_t zero = lds_off(m + (2 * wave + hl) * n + x.reach + kBiasMargin) + 4 * (31 + 8 * hl - j);
    at_m = zero + (qh ? 0 : 64);
    at_q = zero + (qh ? -64 : 128);
  }

  template <int HALF>
  __device__ __forceinline__ void block(const BiasX& x, const float (&ds)[16], int r0) {
    if (r0 > x.reach || r0 + 62 < -x.reach) {
      float t[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) t[i] = (ds[4 * i] + ds[4 * i + 1]) + (ds[4 * i + 2] + ds[4 * i + 3]);
      run[r0 > 0] += (t[0] + t[1]) + (t[2] + t[3]);
      return;
    }
    const uint32_t am = at_m + 4 * (uint32_t)r0, aq = at_q + 4 * (uint32_t)r0;
    uint32_t om = lds_read_b32<0>(am), oq = lds_read_b32<0>(aq);
    float y[2], z[2];
#pragma unroll
    for (int kk = 0; kk < 2; ++kk) {
      y[kk] = ds[8 * kk + 7];
      z[kk] = ds[8 * kk];
    }
#pragma unroll
    for (int e = 1; e < 8; ++e)
#pragma unroll
      for (int kk = 0; kk < 2; ++kk) {
        y[kk] = ds[8 * kk + 7 - e] + dpp<0x101>(y[kk]);  // row_shl:1
        z[kk] = ds[8 * kk + e] + dpp<0x111>(z[kk]);      // row_shr:1
      }
    // rows (qh) of m: distances 16 and 0 ahead of lane j's -j; of y[0]: 0, -16; of z[1]: 32, 16
    float m = y[1] + dpp<0x119>(z[0]);                   // row_shr:9
    const float z1 = dpp<0x119>(z[1]);
    const auto w = __builtin_amdgcn_permlane16_swap(__builtin_bit_cast(uint32_t, z1),
                                                    __builtin_bit_cast(uint32_t, y[0]), false, false);
    // [z1 row 0, y0 row 0] and [z1 row 1, y0 row 1]
    const uint32_t w0 = w[0], w1 = w[1];
    const bool qh = (lane_here() >> 4) & 1;
    m += __builtin_bit_cast(float, qh ? w0 : w1);
    const float q = __builtin_bit_cast(float, qh ? w1 : w0);
    wait_lgkm<0>();
    after_wait(om);
    after_wait(oq);
    lds_write_b32<0>(am, m + __builtin_bit_cast(float, om));
    lds_write_b32<0>(aq, q + __builtin_bit_cast(float, oq));
  }

  // Sums of all waves by distance to out [bias_entries] (all threads; a barrier
  // within). The running sums join their sides' outermost entries, which are of
  // the last bucket, a lane half's in its own array.
  __device__ __forceinline__ void finish(const BiasX& x, float* __restrict__ out, int /*buckets*/, int wave, int waves) {
    const int lane = lane_here(), n = bias_entries(x), hl = lane >> 5;
#pragma unroll
    for (int side = 0; side < 2; ++side) {
      float v = run[side];
#pragma unroll
      for (int m = 16; m >= 1; m >>= 1) v += __shfl_xor(v, m, 64);
      const uint32_t at = lds_off(mem + (2 * wave + hl) * n + (side ? n - 1 : 0));
      uint32_t t = lds_read_b32<0>(at);
      wait_lgkm<0>();
      after_wait(t);
      if ((lane & 31) == 0) lds_write_b32<0>(at, v + __builtin_bit_cast(float, t));
    }
    wait_lgkm<0>();
    __syncthreads();
    for (int e = 64 * wave + lane; e < n; e += 64 * waves) {
      float t = 0.f;
#pragma unroll
      for (int w = 0; w < 2 * waves; ++w) t += mem[w * n + e];
      out[e] = t;
    }
  }
};

// BiasGradWide, where LDS does not hold that: bucket totals of each wave. A block
// of more than one bucket is skewed through LDS, 16 queries at a time: row q of 64
// floats holds key j at column j - q + 15, so a column is a distance; lanes add up
// the columns (lane c: distance r0 + c), a segmented scan joins the lanes of a
// bucket, and its last lane adds the sum to the total.
struct BiasGradWide {
  static constexpr bool kByDistance = false;  // finish's sums are by bucket
  static constexpr int kScratchB = 16 * 64 * 4;
  uint32_t scratch, hist, ids;  // LDS: the wave's rows, its totals; distance 0's bucket id
  float run[2];
  float* totals;

  __host__ __device__ __forceinline__ static int id_bytes(const BiasX& x) { return (bias_entries(x) + 15) / 16 * 16; }
  static size_t lds_bytes(const BiasX& x, int waves) {
    return id_bytes(x) + waves * (kScratchB + 4 * (size_t)x.buckets());
  }

  // (all threads; a barrier must follow)
  template <int HALF>
  __device__ __forceinline__ void init(const BiasX& x, float* m, int buckets, int wave, int waves) {
    const int lane = lane_here();
    unsigned char* id = (unsigned char*)m + waves * kScratchB;
    totals = (float*)(id + id_bytes(x));
    scratch = lds_off((unsigned char*)m + wave * kScratchB);
    hist = lds_off(totals + wave * buckets);
    const int zero = x.reach + kBiasMargin;
    bias_spread(x, 64 * waves, [](int b) CA_INLINE { return b; },
                [&](int e, int b) CA_INLINE { id[e] = (unsigned char)b; });
    if (x.one_sided)  // (keys after their query: masked)
      for (int i = 1 + 64 * wave + lane; i < kBiasMargin; i += 64 * waves) id[zero + i] = 0;
    for (int i = lane; i < buckets; i += 64) totals[wave * buckets + i] = 0.f;
    for (int i = lane; i < kScratchB / 4; i += 64) m[wave * (kScratchB / 4) + i] = 0.f;
    ids = lds_off(id + zero);
    run[0] = run[1] = 0.f;
  }

  __device__ __forceinline__ void add(int id, float v) const {
    uint32_t t = lds_read_b32<0>(hist + 4 * id);
    wait_lgkm<0>();
    after_wait(t);
    lds_write_b32<0>(hist + 4 * id, __builtin_bit_cast(float, t) + v);
  }

  template <int HALF>
  __device__ __forceinline__ void block(const BiasX& x, const float (&ds)[16], int r0) {
    if (r0 > x.reach || r0 + 62 < -x.reach) {
      float t[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) t[i] = (ds[4 * i] + ds[4 * i + 1]) + (ds[4 * i + 2] + ds[4 * i + 3]);
      run[r0 > 0] += (t[0] + t[1]) + (t[2] + t[3]);
      return;
    }
    const int lane = lane_here(), l32 = lane & 31, hl = lane >> 5, row = l32 & 15;
    uint32_t id = lds_read_u8<0>(ids + (uint32_t)(r0 + min(lane, 62)));
    const uint32_t wa = scratch + 4 * (63 * row + 15 + HALF * hl);
    float v = 0.f;
#pragma unroll
    for (int pass = 0; pass < 2; ++pass) {
      if ((l32 >> 4) == pass) {
        auto put = [&](auto i) CA_INLINE {
          constexpr int r = decltype(i)::value, off = HALF == 8 ? 16 * (r >> 3) + (r & 7) : r;
          lds_write_b32<4 * off>(wa, ds[r]);
        };
        for_const<16>(put);
      }
      // queries 0-15 are 16 distances ahead of 16-31 (columns 47-63 are zeros)
      const uint32_t ra = scratch + 4 * (pass == 0 ? (lane + 48) & 63 : lane);
      uint32_t c[16];
      auto get = [&](auto i) CA_INLINE { c[decltype(i)::value] = lds_read_b32<256 * decltype(i)::value>(ra); };
      for_const<16>(get);
      wait_lgkm<0>();
      after_wait(id);
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        after_wait(c[i]);
        v += __builtin_bit_cast(float, c[i]);
      }
    }
#pragma unroll
    for (int s = 1; s < 64; s <<= 1) {
      const float up = __shfl_up(v, s, 64);
      const uint32_t uid = __shfl_up(id, s, 64);
      if (lane >= s && uid == id) v += up;
    }
    const uint32_t next = __shfl_down(id, 1, 64);
    if (lane == 62 || (lane < 62 && next != id)) add(id, v);
  }

  __device__ __forceinline__ void finish(const BiasX& x, float* __restrict__ out, int buckets, int wave, int waves) {
    const int lane = lane_here();
#pragma unroll
    for (int side = 0; side < 2; ++side) {
      float v = run[side];
#pragma unroll
      for (int m = 32; m >= 1; m >>= 1) v += __shfl_xor(v, m, 64);
      if (lane == 0 && !(side && x.one_sided)) add(side ? 2 * x.side - 1 : x.side - 1, v);
    }
    wait_lgkm<0>();
    __syncthreads();
    for (int i = 64 * wave + lane; i < buckets; i += 64 * waves) {
      float t = 0.f;
      for (int w = 0; w < waves; ++w) t += totals[w * buckets + i];
      out[i] = t;
    }
  }
};

// The scale that a bias is divided by: logits are (q.k + bias / s) * s. A scale
// of 0 (or next to it) is taken as 2^-60: q.k s then vanishes beside the bias.
inline float bias_scale(float scale) {
  const float a = __builtin_fabsf(scale);
  return a >= 0x1p-60f ? scale : __builtin_copysignf(0x1p-60f, scale);
}

// Sums of the workgroups' part [B][Hq][n_qt] x [buckets], or x [bias_entries]
// where they are by distance, into dtable (backward.hip).
hipError_t launch_bias_grad(const float* part, bool by_distance, void* dtable, int B, int n_qt, const BiasX& x,
                            hipStream_t stream);

// The device's form of a bias; sizes bound the distances that matter. mul:
// what the kernel's bias is of the table's.
template <class X = BiasX>
inline X bias_x(const EncDecShape& s, const BiasSpec& spec, float eff, float mul) {
  X x;
  x.kv_lens = s.kv_lens;
  x.Skv = s.Skv;
  x.B = s.B;
  x.table = spec.table;
  x.table_dtype = spec.table_dtype;
  x.mul = mul;
  x.scale_log2 = eff * kLog2e;
  x.side = spec.side;
  x.one_sided = spec.one_sided;
  x.Hq = s.Hq;
  for (int i = 0; i < spec.side; ++i) x.first[i] = (uint16_t)spec.first[i];
  x.reach = std::min<int>(spec.first[spec.side - 1], std::max({s.Sq, s.Skv, 1}));
  return x;
}

}  // namespace ca
