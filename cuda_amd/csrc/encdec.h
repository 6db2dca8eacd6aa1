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
// Kernels keep a head's bias by distance in LDS, [-(reach + 96), reach + 95],
// and move a block whose distances all lie past the reach into that margin.
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
};

struct CrossX {
  static constexpr bool kCross = true, kBias = false;
  const int32_t* kv_lens;  // [B], null: Skv for all
  int Skv;
  // keys of sequence b
  __device__ __forceinline__ int kv_len(int b) const {
    const int n = kv_lens ? kv_lens[b] : Skv;
    return __builtin_amdgcn_readfirstlane(min(max(n, 0), Skv));
  }
};

struct BiasX : CrossX {
  static constexpr bool kBias = true;
  const void* table;   // [buckets][Hq] of table_dtype
  int table_dtype;     // kDtypeF32, ...
  float mul;           // table values times this are the kernel's
  float scale_log2;    // ... which, times this, are log2 logits
  int side;            // buckets of a side
  int one_sided;       // keys after their query: distance 0
  int reach;           // distances from here on are in a side's last bucket
  int Hq;
  uint16_t first[kMaxBuckets];  // first distance of a side's bucket
  __device__ __forceinline__ float value(int bucket, int h) const;
};

// ---------------------------------------------------------------------------
// A head's bias by distance in LDS (dynamic: bias_lds_bytes)
// ---------------------------------------------------------------------------
__host__ __device__ constexpr int bias_entries(int reach) { return 2 * reach + 2 * kBiasMargin; }
// the search table, the entries
constexpr int kBiasSearchB = 2 * kMaxBuckets;
constexpr size_t bias_lds_bytes(int reach) { return kBiasSearchB + 4 * (size_t)bias_entries(reach); }

// bucket of distance rel, `first` in LDS
__device__ __forceinline__ int bias_bucket(const BiasX& x, const uint16_t* first, int rel) {
  const int n = rel <= 0 ? -rel : x.one_sided ? 0 : rel;
  int b = 0;
  for (int s = 1 << (31 - __builtin_clz(x.side)); s > 0; s >>= 1)
    if (b + s < x.side && (int)first[b + s] <= n) b += s;
  return b + (rel > 0 && !x.one_sided ? x.side : 0);
}

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

// Fills the workgroup's bias of head h at `mem` (all threads; ends with a
// barrier). Returns the LDS byte offset of distance 0's entry.
__device__ __forceinline__ uint32_t bias_fill(const BiasX& x, int h, unsigned char* mem, int threads) {
  uint16_t* first = (uint16_t*)mem;
  float* e = (float*)(mem + kBiasSearchB);
  // (not from the work-item id, which would stay in a register up to here)
  const int tid = 64 * __builtin_amdgcn_readfirstlane(threadIdx.x >> 6) + lane_here();
  for (int i = tid; i < x.side; i += threads) first[i] = x.first[i];
  __syncthreads();
  const int zero = x.reach + kBiasMargin;
  for (int i = tid; i < bias_entries(x.reach); i += threads)
    e[i] = x.value(bias_bucket(x, first, i - zero), h);
  __syncthreads();
  return lds_off(e + zero);
}

// Distance 0's entry in what bias_fill has filled.
__device__ __forceinline__ const float* bias_zero(const BiasX& x, const unsigned char* mem) {
  return (const float*)(mem + kBiasSearchB) + x.reach + kBiasMargin;
}

// First distance of a block of distances [r0, r0 + 94], moved into the margin
// where all of them lie past the reach.
__device__ __forceinline__ int bias_block(const BiasX& x, int r0) {
  return min(max(r0, -(x.reach + kBiasMargin - 1)), x.reach + 1);
}

// With the ids of the distances' buckets, and the totals of `waves` waves.
constexpr int bias_id_bytes(int reach) { return (bias_entries(reach) + 15) / 16 * 16; }
constexpr size_t bias_grad_lds_bytes(int reach, int buckets, int waves) {
  return bias_lds_bytes(reach) + bias_id_bytes(reach) + 4 * (size_t)buckets * waves;
}

// Ids of the distances' buckets in LDS, beside the entries (all threads; a
// barrier must follow). Returns the byte offset of distance 0's id.
__device__ __forceinline__ uint32_t bias_fill_ids(const BiasX& x, const unsigned char* mem, unsigned char* ids,
                                                  int threads) {
  const int zero = x.reach + kBiasMargin;
  for (int i = threadIdx.x; i < bias_entries(x.reach); i += threads)
    ids[i] = (unsigned char)bias_bucket(x, (const uint16_t*)mem, i - zero);
  return lds_off(ids + zero);
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
  return kBiasSearchB + 64 * (size_t)side + (size_t)(reach + 16) / 16 * 16;
}
// All threads; ends with a barrier. Heads h0 .. h0 + n_heads - 1; the lane's is l16.
__device__ __forceinline__ DecodeBias decode_bias_fill(const BiasX& x, int h0, int n_heads, unsigned char* mem,
                                                       int threads, int l16) {
  uint16_t* first = (uint16_t*)mem;
  float* col = (float*)(mem + kBiasSearchB);
  unsigned char* ids = (unsigned char*)(col + 16 * x.side);
  const int tid = threadIdx.x;
  for (int i = tid; i < x.side; i += threads) first[i] = x.first[i];
  for (int i = tid; i < 16 * x.side; i += threads)
    col[i] = (i & 15) < n_heads ? x.value(i >> 4, h0 + (i & 15)) : 0.f;
  __syncthreads();
  for (int i = tid; i <= x.reach; i += threads) ids[i] = (unsigned char)bias_bucket(x, first, -i);
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
// The table's gradient: sums of dS by bucket, of one wave
// ---------------------------------------------------------------------------
// A 32 x 32 block of dS (lane l32: query, 16 registers: keys) goes to the
// buckets of its 63 distances. Where they are all one bucket, each lane adds its
// registers to a running sum, which is joined when the bucket changes. Otherwise
// the block is skewed through LDS, 16 queries at a time: row q of 64 floats holds
// key j at column j - q + 15, so a column is a distance; lanes add up the columns
// (lane c: distance r0 + c), a segmented scan joins the lanes of a bucket, and
// its last lane adds the sum to the wave's total. No atomics: every total has one
// writer at a time, in program order.
// LDS accesses are hand-issued: the compiler would wait for the tile loads in
// flight before its own.
struct BiasGrad {
  static constexpr int kScratchB = 16 * 64 * 4;
  uint32_t scratch, hist;  // LDS byte offsets: the wave's rows, its totals
  float run;               // the lane's part of the current bucket's sum
  int run_id;

  // zeroes the wave's totals and rows (`scratch_mem`, kScratchB)
  __device__ __forceinline__ void init(uint32_t scratch_mem, uint32_t hist_mem, int buckets) {
    scratch = scratch_mem;
    hist = hist_mem;
    run = 0.f;
    run_id = 0;
    const int lane = lane_here();
    for (int i = lane; i < buckets; i += 64) lds_write_b32<0>(hist + 4 * i, 0.f);
#pragma unroll
    for (int i = 0; i < 16; ++i) lds_write_b32<0>(scratch + 4 * (64 * i + lane), 0.f);
    wait_lgkm<0>();
  }

  __device__ __forceinline__ void add(int id, float v) const {
    uint32_t t = lds_read_b32<0>(hist + 4 * id);
    wait_lgkm<0>();
    after_wait(t);
    lds_write_b32<0>(hist + 4 * id, __builtin_bit_cast(float, t) + v);
  }

  __device__ __forceinline__ void flush() {
    float v = run;
#pragma unroll
    for (int m = 32; m >= 1; m >>= 1) v += __shfl_xor(v, m, 64);
    if (lane_here() == 0) add(run_id, v);
    run = 0.f;
  }

  // The block's dS; register r of half hl is key HALF hl + off(r): HALF = 8, off =
  // 16 (r / 8) + r % 8, or HALF = 16, off = r. `id`: the bucket of distance r0 +
  // min(lane, 62).
  template <int HALF>
  __device__ __forceinline__ void block(const float (&ds)[16], int id) {
    const int id0 = __builtin_amdgcn_readlane(id, 0), id1 = __builtin_amdgcn_readlane(id, 62);
    if (id0 == id1) {
      if (id0 != run_id) {
        flush();
        run_id = id0;
      }
      float t[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) t[i] = (ds[4 * i] + ds[4 * i + 1]) + (ds[4 * i + 2] + ds[4 * i + 3]);
      run += (t[0] + t[1]) + (t[2] + t[3]);
      return;
    }
    const int lane = lane_here(), l32 = lane & 31, hl = lane >> 5, row = l32 & 15;
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
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        after_wait(c[i]);
        v += __builtin_bit_cast(float, c[i]);
      }
    }
#pragma unroll
    for (int s = 1; s < 64; s <<= 1) {
      const float up = __shfl_up(v, s, 64);
      const int uid = __shfl_up(id, s, 64);
      if (lane >= s && uid == id) v += up;
    }
    const int next = __shfl_down(id, 1, 64);
    if (lane == 62 || (lane < 62 && next != id)) add(id, v);
  }
};

// The scale that a bias is divided by: logits are (q.k + bias / s) * s. A scale
// of 0 (or next to it) is taken as 2^-60: q.k s then vanishes beside the bias.
inline float bias_scale(float scale) {
  const float a = __builtin_fabsf(scale);
  return a >= 0x1p-60f ? scale : __builtin_copysignf(0x1p-60f, scale);
}

// The device's form of a bias; sizes bound the distances that matter. mul:
// what the kernel's bias is of the table's.
inline BiasX bias_x(const EncDecShape& s, const BiasSpec& spec, float eff, float mul) {
  BiasX x;
  x.kv_lens = s.kv_lens;
  x.Skv = s.Skv;
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
