// float32 flash-attention backward for gfx950 on fp32 MFMAs.
//
// The reference instantiates its backward for float as well
// (flash_attention_bwd_instantiations.cu:4; binding fused_softmax_binding.cpp:
// 396). Same contract and math as the 16-bit kernels of backward.hip
// (flash_attention_bwd_kernel.cuh:9-19,96-214): from q, k, v, o, dO and the
// forward's natural-log LSE,
//   D_i = rowsum(dO * O),  P = exp(S * scale - LSE_i),  dS = P (dP - D_i),
//   dQ = scale * dS K,  dK = scale * dS^T Q,  dV = P^T dO,
// P = dS = 0 where masked (key > query when causal) or past S; GQA sums dK,
// dV over the q heads of a kv head. Three launches, no atomics.
//
// On v_mfma_f32_32x32x2_f32 (one fp32 element of each operand per lane,
// k = lane / 32), with the float32 forward's row permutation: the A-operand
// lane of output row m reads tile row krow(m) = 16 ((m/4) % 2) + 4 (m/8) +
// m % 4, so accumulator register r of lane half h holds tile row 16 h + r —
// exactly the B-operand element of step r of the next product (which
// contracts tile rows r and 16 + r). P and dS never leave their registers.
//   dq kernel  (4 waves x 32 queries, K/V tiles of 32 keys in LDS):
//     S^T = K Q^T, dP^T = V dO^T, dQ^T += K^T dS^T (K^T read as single
//     floats, 32 consecutive dims per half wave);
//   dkv kernel (4 waves x 32 keys, Q/dO tiles of 32 queries of every q head):
//     S = Q K^T, dP = dO V^T, dV^T += dO^T P, dK^T += Q^T dS.
// Rows are stored with stride D + 4 floats so the float4 row reads of a
// 16-lane group fall on distinct 4-bank groups.
//
// With an X of their own (encdec.h) the same kernels are the backward of cross
// attention and of attention with a relative position bias, which here is added
// to the log2 logits; the dq kernel also sums dS by bucket. Launches of few tiles
// take their SPLIT form: a workgroup has 32 rows (queries, or keys), each wave
// every fourth tile of their walk, staged in LDS of its own (no barriers), and
// the waves add up at the end (2 x 8 heads x 300 queries x 1024 keys x 64: dQ
// 120 -> 38 us, dK/dV 58 -> 46). Where both are SPLIT they are one launch, which
// fills the CUs that either leaves idle (whole backward of the same, with two
// workgroups a CU, 79 -> 69 us; 2 x 12 heads x 500 x 500 with a bias 114 -> 86; 8 / 2
// heads x 700 x 700 182 -> 141).
#include <algorithm>

#include "common.h"
#include "encdec.h"
#include "launch.h"

namespace ca {
namespace {

constexpr int kF32Waves = 4;
constexpr int kF32Tile = 32;

__device__ __forceinline__ int krow32(int l32) {
  return 16 * ((l32 >> 2) & 1) + 4 * (l32 >> 3) + (l32 & 3);
}

// (LSE log2 e, rowsum(dO * O)) per query row; D / 4 lanes per row. X: +inf for
// the LSE of a row without a key, with which every P is 0.
template <int D, class X>
__global__ __launch_bounds__(256) void bwd_rowdot_f32_kernel(const float* __restrict__ O,
                                                             const float* __restrict__ dO,
                                                             const float* __restrict__ LSE,
                                                             float* __restrict__ LD,
                                                             long long rows) {
  constexpr int L = D / 4;
  const long long t = (long long)blockIdx.x * 256 + threadIdx.x;
  const long long row = t / L;
  const int c = (int)(t % L);
  float acc = 0.f;
  if (row < rows) {
    const float4 o = *(const float4*)(O + row * D + 4 * c);
    const float4 g = *(const float4*)(dO + row * D + 4 * c);
    acc = o.x * g.x + o.y * g.y + o.z * g.z + o.w * g.w;
  }
#pragma unroll
  for (int m = L / 2; m >= 1; m >>= 1) acc += __shfl_xor(acc, m, 64);
  if (row < rows && c == 0) {
    const float l = LSE[row];
    LD[2 * row] = X::kCross && l == kNegInf ? -kNegInf : l * kLog2e;
    LD[2 * row + 1] = acc;
  }
}

// Stage 32 rows of two [.., D] fp32 tensors into registers (rows past S as
// zeros), then into padded LDS tiles.
// (T threads: the workgroup's, or a wave's)
template <int D, int T = kF32Waves * 64>
struct Stage2 {
  static constexpr int KS = D + 4;
  static constexpr int F4_ROW = D / 4;
  static constexpr int PER = kF32Tile * F4_ROW / T;
  static_assert(PER * T == kF32Tile * F4_ROW, "staging must cover the tile");
  float4 a[PER], b[PER];
  __device__ __forceinline__ void load(const float* A, const float* B, int r0, int S, int tid) {
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      const int idx = tid + T * i;
      const int row = idx / F4_ROW, c4 = idx % F4_ROW;
      if (r0 + row < S) {
        a[i] = *(const float4*)(A + (size_t)(r0 + row) * D + 4 * c4);
        b[i] = *(const float4*)(B + (size_t)(r0 + row) * D + 4 * c4);
      } else {
        a[i] = float4{0.f, 0.f, 0.f, 0.f};
        b[i] = float4{0.f, 0.f, 0.f, 0.f};
      }
    }
  }
  __device__ __forceinline__ void store(float* As, float* Bs, int tid) const {
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      const int idx = tid + T * i;
      const int row = idx / F4_ROW, c4 = idx % F4_ROW;
      *(float4*)(As + row * KS + 4 * c4) = a[i];
      *(float4*)(Bs + row * KS + 4 * c4) = b[i];
    }
  }
};

// Transposed-accumulator store: acc[ob] rows d = 32 ob + 8 a + 4 h + 0..3,
// column = this lane's row.
template <int NOB>
__device__ __forceinline__ void store_rowT_f32(float* dst_row, const f32x16 (&acc)[NOB], int hl,
                                               float mul) {
#pragma unroll
  for (int ob = 0; ob < NOB; ++ob)
#pragma unroll
    for (int a = 0; a < 4; ++a) {
      const float4 w = {acc[ob][4 * a] * mul, acc[ob][4 * a + 1] * mul, acc[ob][4 * a + 2] * mul,
                        acc[ob][4 * a + 3] * mul};
      *(float4*)(dst_row + 32 * ob + 8 * a + 4 * hl) = w;
    }
}

// A wave's LDS accesses up to here are done before those that follow (its lanes
// read what others of its lanes wrote).
__device__ __forceinline__ void wave_sync() {
  __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
  __builtin_amdgcn_wave_barrier();
  __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
}

// SPLIT: the waves' accumulators added up into wave 0, through LDS at `mem`
// (3 waves' registers, no longer in use as tiles).
template <int N>
__device__ __forceinline__ void sum_waves(f32x16 (&acc)[N], float* mem, int wave, int lane) {
  __syncthreads();
  float4* blk = (float4*)mem + lane;
  if (wave > 0) {
#pragma unroll
    for (int i = 0; i < N; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j)
        blk[64 * (4 * (N * (wave - 1) + i) + j)] =
            float4{acc[i][4 * j], acc[i][4 * j + 1], acc[i][4 * j + 2], acc[i][4 * j + 3]};
  }
  __syncthreads();
  if (wave == 0) {
#pragma unroll
    for (int w = 0; w < kF32Waves - 1; ++w)
#pragma unroll
      for (int i = 0; i < N; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const float4 y = blk[64 * (4 * (N * w + i) + j)];
          acc[i][4 * j] += y.x;
          acc[i][4 * j + 1] += y.y;
          acc[i][4 * j + 2] += y.z;
          acc[i][4 * j + 3] += y.w;
        }
  }
}

// Waves a SIMD: two of SPLIT at head dim 64, which then fit 256 registers (4 x 16
// heads x 200 queries x 700 keys: 136 -> 106 us; with a bias, which takes more of
// them, no gain).
template <int D, class X, bool SPLIT>
constexpr int kF32PerSimd = SPLIT && D == 64 && !X::kBias ? 2 : 1;

// LDS of a workgroup: tiles of two tensors and their rows' (LSE log2 e, D) pairs,
// two in turn (SPLIT: each wave's own).
template <int D, bool SPLIT>
using F32Tiles = float[SPLIT ? kF32Waves : 2][kF32Tile * (D + 4)];
template <bool SPLIT>
using F32Pairs = float[SPLIT ? kF32Waves : 2][2 * kF32Tile];

// dQ: one workgroup = 128 queries of one (b, h) (SPLIT: 32). With a bias, the
// sums of dS by bucket go to part_table [b, h][tile][buckets].
template <int D, bool CAUSAL, class X, bool SPLIT>
__device__ CA_INLINE void bwd_dq_f32_tile(
    const float* Q, const float* K, const float* V,
    const float* dO, const float* LD, float* dQ, int S,
    int Hq, int Hkv, float scale, int n_qt, int block, int n_work, const X& x, float* part_table,
    F32Tiles<D, SPLIT>& Ks, F32Tiles<D, SPLIT>& Vs, unsigned char* bias_mem) {
  constexpr int BM = SPLIT ? 32 : 32 * kF32Waves;
  constexpr int HD = D / 2, NOB = D / 32;
  using St = Stage2<D, SPLIT ? 64 : kF32Waves * 64>;
  constexpr int KS = St::KS;

  const int work = xcd_remap(block, n_work);
  int bh = work / n_qt;
  if constexpr (X::kCross) bh = x.head(bh, Hq).bh;
  const int qt = n_qt - 1 - (work % n_qt);  // longest causal walks first
  const int b = bh / Hq, h = bh % Hq;
  const int hk = h / (Hq / Hkv);
  const int q0 = qt * BM;
  int Skv = S, n_keys = S;
  if constexpr (X::kCross) {
    Skv = x.Skv;
    n_keys = x.kv_len(b);
  }
  const size_t qoff = (size_t)(b * Hq + h) * S;
  const float* Kp = K + (size_t)(b * Hkv + hk) * Skv * D;
  const float* Vp = V + (size_t)(b * Hkv + hk) * Skv * D;

  const int tid = threadIdx.x;
  const int wave = tid >> 6, lane = tid & 63;
  const int l32 = lane & 31, hl = lane >> 5;
  const int qw0 = SPLIT ? q0 : q0 + 32 * wave;
  const int myq = qw0 + l32;
  const bool qvalid = myq < S;
  const float c2 = scale * kLog2e;
  const float lse2 = qvalid ? LD[2 * (qoff + myq)] : -kNegInf;  // past S: P = 0
  const float dd = qvalid ? LD[2 * (qoff + myq) + 1] : 0.f;

  float qv[HD], gv[HD];  // Q and dO as B operands: element HD * hl + k
#pragma unroll
  for (int k4 = 0; k4 < HD; k4 += 4) {
    float4 x = {0.f, 0.f, 0.f, 0.f}, y = {0.f, 0.f, 0.f, 0.f};
    if (qvalid) {
      x = *(const float4*)(Q + (qoff + myq) * D + HD * hl + k4);
      y = *(const float4*)(dO + (qoff + myq) * D + HD * hl + k4);
    }
    qv[k4] = x.x; qv[k4 + 1] = x.y; qv[k4 + 2] = x.z; qv[k4 + 3] = x.w;
    gv[k4] = y.x; gv[k4 + 1] = y.y; gv[k4 + 2] = y.z; gv[k4 + 3] = y.w;
  }

  const float* be = nullptr;  // distance 0's bias, at the lane's query and its first key of a block
  BiasGradWide grad;
  int n_buckets = 0;
  if constexpr (X::kBias) {
    n_buckets = x.buckets();
    grad.init<16>(x, (float*)(bias_mem + bias_lds_bytes(x)), n_buckets, wave, kF32Waves);
    bias_fill<false>(x, h, bias_mem, 64 * kF32Waves);
    be = bias_zero(x, bias_mem) + 31 - l32 + 16 * hl;
  }

  const int kv_end = CAUSAL ? min(n_keys, q0 + BM) : n_keys;
  const int n_tiles = (kv_end + kF32Tile - 1) / kF32Tile;
  St st;
  f32x16 acc[NOB];  // dQ^T
#pragma unroll
  for (int i = 0; i < NOB; ++i)
#pragma unroll
    for (int r = 0; r < 16; ++r) acc[i][r] = 0.f;
  const int krow = krow32(l32);

  const int sid = SPLIT ? lane : tid;               // thread of the staging
  const int t_first = SPLIT ? wave : 0, t_step = SPLIT ? kF32Waves : 1;
  if (t_first < n_tiles) st.load(Kp, Vp, t_first * kF32Tile, n_keys, sid);
  for (int t = t_first; t < n_tiles; t += t_step) {
    const int buf = SPLIT ? wave : t & 1;
    if constexpr (SPLIT) wave_sync();  // the tile before has been read
    st.store(Ks[buf], Vs[buf], sid);
    if constexpr (SPLIT) wave_sync();
    else __syncthreads();
    if (t + t_step < n_tiles) st.load(Kp, Vp, (t + t_step) * kF32Tile, n_keys, sid);
    const int k0 = t * kF32Tile;
    if (CAUSAL && k0 > qw0 + 31) continue;  // every key after every query of the wave
    // S^T = K Q^T, dP^T = V dO^T; register r of half hl <-> key k0 + 16 hl + r
    f32x16 s, dp;
#pragma unroll
    for (int r = 0; r < 16; ++r) { s[r] = 0.f; dp[r] = 0.f; }
    const float* kr = Ks[buf] + krow * KS + HD * hl;
    const float* vr = Vs[buf] + krow * KS + HD * hl;
#pragma unroll
    for (int k4 = 0; k4 < HD; k4 += 4) {
      const float4 a = *(const float4*)(kr + k4);
      const float4 c = *(const float4*)(vr + k4);
      s = __builtin_amdgcn_mfma_f32_32x32x2f32(a.x, qv[k4], s, 0, 0, 0);
      dp = __builtin_amdgcn_mfma_f32_32x32x2f32(c.x, gv[k4], dp, 0, 0, 0);
      s = __builtin_amdgcn_mfma_f32_32x32x2f32(a.y, qv[k4 + 1], s, 0, 0, 0);
      dp = __builtin_amdgcn_mfma_f32_32x32x2f32(c.y, gv[k4 + 1], dp, 0, 0, 0);
      s = __builtin_amdgcn_mfma_f32_32x32x2f32(a.z, qv[k4 + 2], s, 0, 0, 0);
      dp = __builtin_amdgcn_mfma_f32_32x32x2f32(c.z, gv[k4 + 2], dp, 0, 0, 0);
      s = __builtin_amdgcn_mfma_f32_32x32x2f32(a.w, qv[k4 + 3], s, 0, 0, 0);
      dp = __builtin_amdgcn_mfma_f32_32x32x2f32(c.w, gv[k4 + 3], dp, 0, 0, 0);
    }
    const bool need_mask =
        CAUSAL ? (k0 + kF32Tile - 1 > qw0 || (X::kCross && k0 + kF32Tile > n_keys)) : (k0 + kF32Tile > n_keys);
    float ds[16];  // dS^T / scale
    const float* bb = be;
    if constexpr (X::kBias) bb += bias_block(x, k0 - qw0 - 31);
#pragma unroll
    for (int r = 0; r < 16; ++r) {
      float e = __builtin_fmaf(s[r], c2, -lse2);
      if constexpr (X::kBias) e += bb[r];
      float p = fast_exp2(e);
      if (need_mask) {
        const int key = k0 + 16 * hl + r;
        if (key >= n_keys || (CAUSAL && key > myq)) p = 0.f;
      }
      ds[r] = p * (dp[r] - dd);
    }
    // dQ^T[d x q] += K^T[d x keys] dS^T[keys x q]: step r contracts keys r, 16 + r
#pragma unroll
    for (int ob = 0; ob < NOB; ++ob) {
      const float* kt = Ks[buf] + (16 * hl) * KS + 32 * ob + l32;
#pragma unroll
      for (int r = 0; r < 16; ++r)
        acc[ob] = __builtin_amdgcn_mfma_f32_32x32x2f32(kt[r * KS], ds[r], acc[ob], 0, 0, 0);
    }
    if constexpr (X::kBias) grad.template block<16>(x, ds, k0 - qw0 - 31);
  }
  if constexpr (X::kBias)
    grad.finish(x, part_table + ((size_t)bh * n_qt + qt) * n_buckets, n_buckets, wave, kF32Waves);
  if constexpr (SPLIT) {
    sum_waves<NOB>(acc, Ks[0], wave, lane);
    if (wave > 0) return;
  }
  if (qvalid) store_rowT_f32<NOB>(dQ + (qoff + myq) * D, acc, hl, scale);
}

template <int D, bool CAUSAL, class X, bool SPLIT>
__global__ __launch_bounds__(kF32Waves * 64, (kF32PerSimd<D, X, SPLIT>)) void bwd_dq_f32_kernel(
    const float* __restrict__ Q, const float* __restrict__ K, const float* __restrict__ V,
    const float* __restrict__ dO, const float* __restrict__ LD, float* __restrict__ dQ, int S,
    int Hq, int Hkv, float scale, int n_qt, int n_work, X x, float* __restrict__ part_table) {
  extern __shared__ __attribute__((aligned(16))) unsigned char bias_mem[];
  __shared__ __attribute__((aligned(16))) F32Tiles<D, SPLIT> Ks, Vs;
  bwd_dq_f32_tile<D, CAUSAL, X, SPLIT>(Q, K, V, dO, LD, dQ, S, Hq, Hkv, scale, n_qt, blockIdx.x, n_work, x,
                                       part_table, Ks, Vs, bias_mem);
}

// dK, dV: one workgroup = 128 keys of one (b, kv head) (SPLIT: 32); 32-query tiles
// of every q head of the kv head.
template <int D, bool CAUSAL, class X, bool SPLIT>
__device__ CA_INLINE void bwd_dkv_f32_tile(
    const float* Q, const float* K, const float* V,
    const float* dO, const float* LD, float* dK,
    float* dV, int S, int Hq, int Hkv, float scale, int n_kt, int block, int n_work, const X& x,
    F32Tiles<D, SPLIT>& Qs, F32Tiles<D, SPLIT>& Gs, F32Pairs<SPLIT>& Ls, unsigned char* bias_mem) {
  constexpr int BK = SPLIT ? 32 : 32 * kF32Waves;
  constexpr int HD = D / 2, NOB = D / 32;
  using St = Stage2<D, SPLIT ? 64 : kF32Waves * 64>;
  constexpr int KS = St::KS;

  const int work = xcd_remap(block, n_work);
  int bhk = work / n_kt;
  if constexpr (X::kCross) bhk = x.head(bhk, Hkv).bh;
  const int kt = work % n_kt;  // causal: the first key tiles have the longest query walks
  const int b = bhk / Hkv, hk = bhk % Hkv;
  const int G = Hq / Hkv;
  const int K0 = kt * BK;
  int Skv = S, n_keys = S;
  if constexpr (X::kCross) {
    Skv = x.Skv;
    n_keys = x.kv_len(b);
  }
  const size_t kvoff = (size_t)(b * Hkv + hk) * Skv;

  const int tid = threadIdx.x;
  const int wave = tid >> 6, lane = tid & 63;
  const int l32 = lane & 31, hl = lane >> 5;
  const int kw0 = SPLIT ? K0 : K0 + 32 * wave;
  const int mykey = kw0 + l32;
  const bool kvalid = mykey < n_keys;
  const float c2 = scale * kLog2e;

  float kv[HD], vv[HD];  // K^T and V^T as B operands: element HD * hl + k of this lane's key
#pragma unroll
  for (int k4 = 0; k4 < HD; k4 += 4) {
    float4 x = {0.f, 0.f, 0.f, 0.f}, y = {0.f, 0.f, 0.f, 0.f};
    if (kvalid) {
      x = *(const float4*)(K + (kvoff + mykey) * D + HD * hl + k4);
      y = *(const float4*)(V + (kvoff + mykey) * D + HD * hl + k4);
    }
    kv[k4] = x.x; kv[k4 + 1] = x.y; kv[k4 + 2] = x.z; kv[k4 + 3] = x.w;
    vv[k4] = y.x; vv[k4 + 1] = y.y; vv[k4 + 2] = y.z; vv[k4 + 3] = y.w;
  }

  const int t_begin = CAUSAL ? K0 / kF32Tile : 0;
  int nt = max(0, (S + kF32Tile - 1) / kF32Tile - t_begin);
  if constexpr (X::kCross)
    if (K0 >= n_keys) nt = 0;
  const int n_it = G * nt;
  const int sid = SPLIT ? lane : tid;  // thread of the staging
  constexpr int it_step = SPLIT ? kF32Waves : 1;
  St st;
  float lreg = 0.f;
  auto gload = [&](int it) {
    const int hq = hk * G + it / nt;
    const int q0 = (t_begin + it % nt) * kF32Tile;
    const size_t qoff = (size_t)(b * Hq + hq) * S;
    st.load(Q + qoff * D, dO + qoff * D, q0, S, sid);
    if (sid < 2 * kF32Tile) {  // pair element sid of the tile's 32 rows
      const int row = q0 + (sid >> 1);
      lreg = row < S ? LD[2 * (qoff + row) + (sid & 1)] : ((sid & 1) ? 0.f : -kNegInf);
    }
  };

  f32x16 dk[NOB], dv[NOB];
#pragma unroll
  for (int i = 0; i < NOB; ++i)
#pragma unroll
    for (int r = 0; r < 16; ++r) { dk[i][r] = 0.f; dv[i][r] = 0.f; }
  const int qrow = krow32(l32);

  // the next tile is loaded beside this one's products, where there are registers
  // for it (SPLIT stages four times the rows a lane)
  constexpr bool kAhead = !SPLIT || (D == 64 && kF32PerSimd<D, X, SPLIT> == 1);
  // With a bias the walk is one q head's tiles after the other's (LDS holds one
  // head's bias), otherwise all tiles at once.
  int g = 0;
  do {
  int it_first = SPLIT ? wave : 0, it_end = n_it;
  if constexpr (X::kBias) {
    if (nt == 0) break;
    if (g > 0) __syncthreads();  // every wave has read the last head's
    bias_fill<false>(x, hk * G + g, bias_mem, 64 * kF32Waves);
    it_first += g * nt;
    it_end = (g + 1) * nt;
  }
  if (kAhead && it_first < it_end) gload(it_first);
  for (int it = it_first; it < it_end; it += it_step) {
    const int buf = SPLIT ? wave : it & 1;
    if constexpr (!kAhead) gload(it);
    if constexpr (SPLIT) wave_sync();  // the tile before has been read
    st.store(Qs[buf], Gs[buf], sid);
    if (sid < 2 * kF32Tile) Ls[buf][sid] = lreg;
    if constexpr (SPLIT) wave_sync();
    else __syncthreads();
    if (kAhead && it + it_step < it_end) gload(it + it_step);
    const int q0 = (t_begin + it % nt) * kF32Tile;
    if (CAUSAL && q0 + 31 < kw0) continue;  // every query before every key of the wave
    // S = Q K^T, dP = dO V^T; register r of half hl <-> query q0 + 16 hl + r
    f32x16 s, dp;
#pragma unroll
    for (int r = 0; r < 16; ++r) { s[r] = 0.f; dp[r] = 0.f; }
    const float* qr = Qs[buf] + qrow * KS + HD * hl;
    const float* gr = Gs[buf] + qrow * KS + HD * hl;
#pragma unroll
    for (int k4 = 0; k4 < HD; k4 += 4) {
      const float4 a = *(const float4*)(qr + k4);
      const float4 c = *(const float4*)(gr + k4);
      s = __builtin_amdgcn_mfma_f32_32x32x2f32(a.x, kv[k4], s, 0, 0, 0);
      dp = __builtin_amdgcn_mfma_f32_32x32x2f32(c.x, vv[k4], dp, 0, 0, 0);
      s = __builtin_amdgcn_mfma_f32_32x32x2f32(a.y, kv[k4 + 1], s, 0, 0, 0);
      dp = __builtin_amdgcn_mfma_f32_32x32x2f32(c.y, vv[k4 + 1], dp, 0, 0, 0);
      s = __builtin_amdgcn_mfma_f32_32x32x2f32(a.z, kv[k4 + 2], s, 0, 0, 0);
      dp = __builtin_amdgcn_mfma_f32_32x32x2f32(c.z, vv[k4 + 2], dp, 0, 0, 0);
      s = __builtin_amdgcn_mfma_f32_32x32x2f32(a.w, kv[k4 + 3], s, 0, 0, 0);
      dp = __builtin_amdgcn_mfma_f32_32x32x2f32(c.w, vv[k4 + 3], dp, 0, 0, 0);
    }
    const bool need_mask = !kvalid || (CAUSAL && q0 < kw0 + 31) || q0 + kF32Tile > S;
    float p[16], ds[16];
    // register r: distance kw0 + l32 - (q0 + 16 hl + r)
    const float* bb = nullptr;
    if constexpr (X::kBias) bb = bias_zero(x, bias_mem) + bias_block(x, kw0 - q0 - 31) + 31 + l32 - 16 * hl;
#pragma unroll
    for (int r = 0; r < 16; ++r) {
      const int qi = 16 * hl + r;
      float e = __builtin_fmaf(s[r], c2, -Ls[buf][2 * qi]);
      if constexpr (X::kBias) e += bb[-r];
      p[r] = fast_exp2(e);
      if (need_mask) {
        const int query = q0 + qi;
        if (!kvalid || query >= S || (CAUSAL && mykey > query)) p[r] = 0.f;
      }
      ds[r] = p[r] * (dp[r] - Ls[buf][2 * qi + 1]);
    }
    // dV^T[d x keys] += dO^T P, dK^T[d x keys] += Q^T dS: step r contracts
    // queries r, 16 + r
#pragma unroll
    for (int ob = 0; ob < NOB; ++ob) {
      const float* gt = Gs[buf] + (16 * hl) * KS + 32 * ob + l32;
      const float* qt = Qs[buf] + (16 * hl) * KS + 32 * ob + l32;
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        dv[ob] = __builtin_amdgcn_mfma_f32_32x32x2f32(gt[r * KS], p[r], dv[ob], 0, 0, 0);
        dk[ob] = __builtin_amdgcn_mfma_f32_32x32x2f32(qt[r * KS], ds[r], dk[ob], 0, 0, 0);
      }
    }
  }
  } while (X::kBias && ++g < G);
  if constexpr (SPLIT) {
    sum_waves<NOB>(dk, Qs[0], wave, lane);
    sum_waves<NOB>(dv, Qs[0], wave, lane);
    if (wave > 0) return;
  }
  if constexpr (X::kCross) {
    if (!kvalid) {  // a padded key: 0
#pragma unroll
      for (int i = 0; i < NOB; ++i)
#pragma unroll
        for (int r = 0; r < 16; ++r) { dk[i][r] = 0.f; dv[i][r] = 0.f; }
    }
  }
  if (mykey < Skv) {
    store_rowT_f32<NOB>(dK + (kvoff + mykey) * D, dk, hl, scale);
    store_rowT_f32<NOB>(dV + (kvoff + mykey) * D, dv, hl, 1.f);
  }
}

template <int D, bool CAUSAL, class X, bool SPLIT>
__global__ __launch_bounds__(kF32Waves * 64, (kF32PerSimd<D, X, SPLIT>)) void bwd_dkv_f32_kernel(
    const float* __restrict__ Q, const float* __restrict__ K, const float* __restrict__ V,
    const float* __restrict__ dO, const float* __restrict__ LD, float* __restrict__ dK,
    float* __restrict__ dV, int S, int Hq, int Hkv, float scale, int n_kt, int n_work, X x) {
  extern __shared__ __attribute__((aligned(16))) unsigned char bias_mem[];
  __shared__ __attribute__((aligned(16))) F32Tiles<D, SPLIT> Qs, Gs;  // Q, dO
  __shared__ __attribute__((aligned(16))) F32Pairs<SPLIT> Ls;
  bwd_dkv_f32_tile<D, CAUSAL, X, SPLIT>(Q, K, V, dO, LD, dK, dV, S, Hq, Hkv, scale, n_kt,
                                        blockIdx.x, n_work, x, Qs, Gs, Ls, bias_mem);
}

// Both in one launch, where both are SPLIT: the workgroups with the longer walks
// first, the others behind them wherever a CU is free.
template <int D, bool CAUSAL, class X>
__global__ __launch_bounds__(kF32Waves * 64, (kF32PerSimd<D, X, true>)) void bwd_both_f32_kernel(
    const float* __restrict__ Q, const float* __restrict__ K, const float* __restrict__ V,
    const float* __restrict__ dO, const float* __restrict__ LD, float* __restrict__ dQ,
    float* __restrict__ dK, float* __restrict__ dV, int S, int Hq, int Hkv, float scale, int n_qt, int n_kt,
    int n_dq, int n_dkv, int dkv_first, X x, float* __restrict__ part_table) {
  extern __shared__ __attribute__((aligned(16))) unsigned char bias_mem[];
  __shared__ __attribute__((aligned(16))) F32Tiles<D, true> As, Bs;
  __shared__ __attribute__((aligned(16))) F32Pairs<true> Ls;
  const int i = blockIdx.x, first = dkv_first ? n_dkv : n_dq;
  if ((i < first) == (dkv_first != 0))
    bwd_dkv_f32_tile<D, CAUSAL, X, true>(Q, K, V, dO, LD, dK, dV, S, Hq, Hkv, scale, n_kt,
                                         dkv_first ? i : i - first, n_dkv, x, As, Bs, Ls, bias_mem);
  else
    bwd_dq_f32_tile<D, CAUSAL, X, true>(Q, K, V, dO, LD, dQ, S, Hq, Hkv, scale, n_qt,
                                        dkv_first ? i - first : i, n_dq, x, part_table, As, Bs, bias_mem);
}

// Whether a launch over `heads` heads of `rows` rows takes 32 rows a workgroup,
// their walk in four parts: where that shortens the busiest CU's work by a fifth,
// and LDS holds the waves' tiles beside what a bias takes.
bool bwd_f32_fits(int D, size_t bias_lds) {
  return kF32Waves * (2 * kF32Tile * (D + 4) + 2 * kF32Tile) * sizeof(float) + bias_lds <= 160 * 1024;
}
bool bwd_f32_splits(long long heads, int rows, int D, size_t bias_lds) {
  if (!bwd_f32_fits(D, bias_lds)) return false;
  const long long cus = device_cus() > 0 ? device_cus() : 1;
  const long long whole = heads * ((rows + 127) / 128), split = heads * ((rows + 31) / 32);
  return 10 * ((split + cus - 1) / cus) < 8 * 4 * ((whole + cus - 1) / cus);
}

template <int D, bool CAUSAL, class X>
hipError_t launch_bwd_f32_t(const float* q, const float* k, const float* v, const float* o,
                            const float* dout, const float* lse, float* dq, float* dk, float* dv,
                            int B, int Hq, int Hkv, int S, int Skv, float scale, float* ws, const X& x,
                            size_t dkv_lds, size_t dq_lds, float* part_table, void* dtable,
                            hipStream_t stream) {
  const long long rows = (long long)B * Hq * S;
  const long long g0 = (rows * (D / 4) + 255) / 256;
  auto dqk = &bwd_dq_f32_kernel<D, CAUSAL, X, false>;
  auto dkvk = &bwd_dkv_f32_kernel<D, CAUSAL, X, false>;
  int bm = 32 * kF32Waves, bk = 32 * kF32Waves;
  if constexpr (X::kCross) {
    if (bwd_f32_splits((long long)B * Hq, S, D, dq_lds)) {
      dqk = &bwd_dq_f32_kernel<D, CAUSAL, X, true>;
      bm = 32;
    }
    if (bwd_f32_splits((long long)B * Hkv, Skv, D, dkv_lds)) {
      dkvk = &bwd_dkv_f32_kernel<D, CAUSAL, X, true>;
      bk = 32;
    }
  }
  const int n_qt = (S + bm - 1) / bm;
  const int n_kt = (Skv + bk - 1) / bk;
  const long long gq = (long long)B * Hq * n_qt;
  const long long gk = (long long)B * Hkv * n_kt;
  if (g0 > 0x7fffffffLL || gq > 0x7fffffffLL || gk > 0x7fffffffLL) return hipErrorInvalidValue;
  hipError_t e = hipSuccess;
  if (g0 > 0) {
    hipLaunchKernelGGL((bwd_rowdot_f32_kernel<D, X>), dim3((unsigned)g0), dim3(256), 0, stream, o, dout,
                       lse, ws, rows);
    e = hipGetLastError();
    if (e != hipSuccess) return e;
  }
  if constexpr (X::kCross) {
    const size_t lds = std::max(dkv_lds, dq_lds);
    if (bm == 32 && bk == 32 && gq + gk <= 0x7fffffffLL && bwd_f32_fits(D, lds)) {
      // (walks in products of a tile: dQ's 3 over the keys, dK/dV's 4 over the kv head's queries)
      const bool dkv_first = 4LL * (Hq / Hkv) * S > 3LL * Skv;
      hipLaunchKernelGGL((bwd_both_f32_kernel<D, CAUSAL, X>), dim3((unsigned)(gq + gk)), dim3(kF32Waves * 64), lds,
                         stream, q, k, v, dout, ws, dq, dk, dv, S, Hq, Hkv, scale, n_qt, n_kt, (int)gq, (int)gk,
                         (int)dkv_first, x, part_table);
      e = hipGetLastError();
      if (e != hipSuccess) return e;
      if constexpr (X::kBias) return launch_bias_grad(part_table, false, dtable, B, n_qt, x, stream);
      return e;
    }
  }
  if (gk > 0) {
    hipLaunchKernelGGL(dkvk, dim3((unsigned)gk), dim3(kF32Waves * 64), dkv_lds,
                       stream, q, k, v, dout, ws, dk, dv, S, Hq, Hkv, scale, n_kt, (int)gk, x);
    e = hipGetLastError();
    if (e != hipSuccess) return e;
  }
  if (gq > 0) {
    hipLaunchKernelGGL(dqk, dim3((unsigned)gq), dim3(kF32Waves * 64), dq_lds,
                       stream, q, k, v, dout, ws, dq, S, Hq, Hkv, scale, n_qt, (int)gq, x, part_table);
    e = hipGetLastError();
    if (e != hipSuccess) return e;
  }
  if constexpr (X::kBias)
    return launch_bias_grad(part_table, false, dtable, B, n_qt, x, stream);
  return e;
}

}  // namespace

hipError_t launch_flash_bwd_f32(const float* q, const float* k, const float* v, const float* o,
                                const float* dout, const float* lse, float* dq, float* dk,
                                float* dv, int B, int Hq, int Hkv, int S, int D, float scale,
                                bool causal, void* ws, hipStream_t stream) {
  if ((long long)B * Hq * S == 0) return hipSuccess;
  float* w = (float*)ws;
  const SelfX x;
#define CA_BWD32(DD, CAUSAL)                                                                                      \
  launch_bwd_f32_t<DD, CAUSAL>(q, k, v, o, dout, lse, dq, dk, dv, B, Hq, Hkv, S, S, scale, w, x, 0, 0, nullptr, \
                               nullptr, stream)
  if (D == 64) return causal ? CA_BWD32(64, true) : CA_BWD32(64, false);
  if (D == 128) return causal ? CA_BWD32(128, true) : CA_BWD32(128, false);
#undef CA_BWD32
  return hipErrorInvalidValue;
}

hipError_t launch_cross_bwd_f32(const float* q, const float* k, const float* v, const float* o, const float* dout,
                                const float* lse, float* dq, float* dk, float* dv, void* dtable,
                                const EncDecShape& s, const BiasSpec* bias, bool causal, float* ws,
                                hipStream_t stream) {
#define CA_BWD32(DD, CAUSAL, X, DKV, DQ, PART)                                                               \
  launch_bwd_f32_t<DD, CAUSAL>(q, k, v, o, dout, lse, dq, dk, dv, s.B, s.Hq, s.Hkv, s.Sq, s.Skv, s.scale, ws, \
                               X, DKV, DQ, PART, dtable, stream)
  if (!bias) {
    CrossX x;
    x.kv_lens = s.kv_lens;
    x.Skv = s.Skv;
    x.B = s.B;
    if (s.D == 64) return CA_BWD32(64, false, x, 0, 0, nullptr);
    if (s.D == 128) return CA_BWD32(128, false, x, 0, 0, nullptr);
    return hipErrorInvalidValue;
  }
  const BiasX x = bias_x(s, *bias, s.scale, kLog2e);
  const size_t dkv = bias_lds_bytes(x);
  const size_t dqb = dkv + BiasGradWide::lds_bytes(x, kF32Waves);
  float* part = ws + 2 * (size_t)s.B * s.Hq * s.Sq;
  if (s.D == 64) return causal ? CA_BWD32(64, true, x, dkv, dqb, part) : CA_BWD32(64, false, x, dkv, dqb, part);
  if (s.D == 128) return causal ? CA_BWD32(128, true, x, dkv, dqb, part) : CA_BWD32(128, false, x, dkv, dqb, part);
#undef CA_BWD32
  return hipErrorInvalidValue;
}

}  // namespace ca
