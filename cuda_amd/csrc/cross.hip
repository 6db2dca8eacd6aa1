// Attention of encoder-decoder models, forward, 16-bit: cross attention (keys of
// another length, padded per sequence) and self-attention with a learned
// relative position bias (encdec.h).
//
// Computes O = softmax(Q K^T * scale [+ bias(key - query)] [+ causal mask]) V
// over the first kv_len keys of each sequence, and the natural-log LSE; a row
// with no key gives 0 and -inf. Math, tiles and register layouts are those of
// prefill_rows.hip: a workgroup takes 32 QG query rows, QG row groups of KS =
// 8 / QG waves ("parts"), each part walking every KS-th key tile with an online
// softmax of its own; the parts meet in LDS. S^T = K Q^T with the rho row
// permutation, whose accumulators are the B operand of O^T += V^T P^T.
//
// Cross attention has no position, and the query rows of the G heads of a kv
// head lie one after the other, so a tile's rows run over all of them: G Sq
// rows of a kv head make as few tiles as they can.
//
// The bias enters as the accumulators' start: S^T begins as bias / scale, so it
// costs LDS reads (two dwords a lane for two logits) and no VALU work.
//
// What bounds it: long walks the matrix pipes with the softmax's VALU beside them.
// bf16, 4 x 32 heads x 2048 queries x 1792 to 4096 keys x 128: 360 us, 1.10 PFLOP/s
// (a large matrix product: 1.24 to 1.39); causal with a bias, 32 heads x 8192 x 64:
// 320 us, 0.85 PFLOP/s (half the products a logit for the same exponential, and the
// bias reads). Short ones the way of the first keys from HBM and the launch: 12
// heads x 100 x 100 x 64 with a bias 7.7 us, of which an empty launch is 4.4.
#include <algorithm>
#include <cmath>
#include <type_traits>

#include "common.h"
#include "encdec.h"
#include "launch.h"
#include "lds_dma.h"
#include "prefill_common.h"

namespace ca {
namespace {

constexpr int kWaves = 8;
template <int D>
constexpr int kStepTiles = D == 64 ? 4 : 2;

struct CrossArgs {
  const uint16_t* q;
  const uint16_t* k;
  const uint16_t* v;
  uint16_t* o;
  uint16_t* o_low;  // what o's rounding took, or null
  float* lse;
  float* part_o;    // [rows of all groups][n_split][D], o / l, where n_split > 1
  float* part_lse;  // ... log2 of the sum of 2^x
  int rows;         // query rows of a group (a head, or a kv head's heads)
  int per_b;        // groups per sequence
  int ratio;        // groups per kv head
  float scale_log2; // |scale| log2 e
  uint32_t q_sign;  // flips q's signs for a negative scale
  int n_qt, n_bh, n_work, order, n_split;
};

// Split `split` of the key walk of query tile qt of group bh.
template <typename Tr, int D, class X, bool CAUSAL, int QG>
__device__ CA_INLINE void cross_tile(const CrossArgs& a, const X& x, unsigned char* bias_mem, int bh, int n_keys,
                                     int qt, int split) {
  using Gm = PfGeom<D>;
  using vec8 = typename Tr::vec8;
  using vec4 = typename Tr::vec4;
  using vec2 = typename Tr::vec2;
  constexpr bool BIAS = X::kBias;
  constexpr int kNW = kWaves, KS = kNW / QG;
  // 64 keys per tile; 32 where four 64-key tiles would fill the ring
  constexpr int kBN = D == 128 && KS == 4 ? 32 : 64;
  constexpr int kMB = kBN / 32;                  // 32-key blocks per tile
  constexpr int kKK = kBN / 16;                  // PV k-steps per tile
  constexpr int kRowB = Gm::kRowB, kNKS = Gm::kNKS, kNOB = Gm::kNOB;
  constexpr int kTileB = kBN * kRowB;            // K (or V) tile
  // key tiles per part and barrier: a SIMD's two waves may drift apart by that many
  constexpr int NT = KS == 1 ? kStepTiles<D> : 1;
  constexpr int kGroupB = KS * NT * 2 * kTileB;  // NT K and V tiles per part
  constexpr int kGroups = 128 * 1024 / kGroupB;  // ring, groups
  static_assert(kGroups >= 2, "a group loads while another is read");
  constexpr int kT = kTileB / 1024;              // 1-KB loads per tile
  constexpr int kLoads = KS * NT * 2 * kT / kNW; // loads per wave per group
  static_assert(kT % kNW == 0, "a tile's loads are dealt to all waves");
  constexpr int NR = 16 * kNOB / KS;             // O^T registers a part combines
  constexpr int kMeetB = QG * KS * (KS - 1) * NR * 256;  // the others' registers
  constexpr int kRowsB = QG * 32 * kRowB;        // output rows, packed
  static_assert(kMeetB + kRowsB <= kGroups * kGroupB, "the meeting fits the ring");
  __shared__ __attribute__((aligned(1024))) unsigned char lds[kGroups * kGroupB];
  __shared__ float red_m[QG][KS][32], red_l[QG][KS][32];

  const int rows = a.rows;
  const int lane = lane_here();  // (not hoisted out of the pair's loop: registers)
  const int wave = __builtin_amdgcn_readfirstlane(__builtin_amdgcn_workitem_id_x() >> 6);
  const int qg = wave % QG, part = wave / QG;
  const int l32 = lane & 31, hl = lane >> 5;
  const int q0 = qt * 32 * QG, qw0 = q0 + 32 * qg, myq = qw0 + l32;
  const bool q_in = myq < rows;
  const int b = bh / a.per_b, g_in_b = bh % a.per_b;
  const size_t khead = ((size_t)b * (a.per_b / a.ratio) + g_in_b / a.ratio) * x.Skv;
  const uint16_t* Kp = a.k + khead * D;
  const uint16_t* Vp = a.v + khead * D;

  const int kv_end = CAUSAL ? min(n_keys, q0 + 32 * QG) : n_keys;
  const int n_all = (kv_end + kBN - 1) / kBN;
  // this split's tiles [t0, t0 + n_tiles)
  const int t0 = (int)((long long)n_all * split / a.n_split);
  const int n_tiles = (int)((long long)n_all * (split + 1) / a.n_split) - t0;
  const int n_groups = (n_tiles + KS * NT - 1) / (KS * NT);
  // tiles this row group computes; the last of the whole walk holds the
  // diagonal or the end
  const int w_end = CAUSAL ? min(kv_end, qw0 + 32) : kv_end;
  const int w_last = (w_end + kBN - 1) / kBN - 1 - t0;
  const int w_tiles = qw0 < rows ? min(w_last + 1, n_tiles) : 0;

  // load j of this wave: 1 KB of tile `sub` of the group, K or V, rows from
  // kRpk * piece (rows past kv_end read as zero)
  uint32_t off0;
  {
    const int row = Gm::kRpk * wave + lane / Gm::kLpr;
    off0 = row * kRowB + 16 * ((lane % Gm::kLpr) ^ Gm::swz(row));
  }
  // load j of the group's tile `sub`: K loads, then V loads
  constexpr int kPer = kT / kNW;  // loads of a wave per tile, of K and of V
  auto issue_one = [&](int g, int sub, int j) CA_INLINE {
    const int is_v = j / kPer, p = j % kPer;
    const uint32_t t = (uint32_t)(t0 + g * KS * NT + sub);
    dma16_buf(make_rsrc_at(is_v ? Vp : Kp, t * kTileB, (uint32_t)kv_end * kRowB),
              (CA_LDS void*)(lds + (g % kGroups) * kGroupB + (2 * sub + is_v) * kTileB + 1024 * (kNW * p + wave)),
              off0 + 1024u * kNW * p);  // swz repeats every 16 rows
  };
  auto issue = [&](int g) CA_INLINE {
#pragma unroll
    for (int sub = 0; sub < KS * NT; ++sub)
#pragma unroll
      for (int j = 0; j < 2 * kPer; ++j) issue_one(g, sub, j);
  };
#pragma unroll
  for (int g = 0; g < kGroups - 1; ++g) issue(g);

  // Q as the B operand of S^T = K Q^T: k-step ks holds d = 16 ks + 8 hl + [0, 8).
  // Lanes past the rows take the last one.
  vec8 qv[kNKS];
  {
    const uint16_t* Qr = a.q + ((size_t)bh * rows + min(myq, rows - 1)) * D;
#pragma unroll
    for (int ks = 0; ks < kNKS; ++ks) {
      u32x4 w = *(const u32x4*)(Qr + 16 * ks + 8 * hl);
      w ^= a.q_sign;
      qv[ks] = __builtin_bit_cast(vec8, w);
    }
  }

  // LDS read offsets (prefill.hip): K row rho(l32), chunk hl (^ 32 ks bytes);
  // V^T source rows tr_row and tr_row + 4, chunks c0 (^ 64 ob bytes)
  const int krow = (l32 & 0x13) | ((l32 & 4) << 1) | ((l32 & 8) >> 1);
  const uint32_t kofs = krow * kRowB + 16 * (hl ^ Gm::swz(krow));
  const int g16 = lane >> 4, s16 = lane & 15;
  const int tr_row = 8 * (g16 >> 1) + (s16 >> 2), c0 = 2 * (g16 & 1) + ((s16 & 3) >> 1);
  const uint32_t vofs1 = kTileB + tr_row * kRowB + 16 * (c0 ^ Gm::swz(tr_row)) + 8 * (s16 & 1);
  const uint32_t vofs2 =
      kTileB + (tr_row + 4) * kRowB + 16 * (c0 ^ Gm::swz(tr_row + 4)) + 8 * (s16 & 1);
  const uint32_t lds0 = lds_off(lds);
  // the bias of the lane's query and its first key of a block that starts at
  // distance r0: register i is 4 (31 - l32 + 8 hl + off(i)) bytes past entry r0
  uint32_t bofs = 0;
  if constexpr (BIAS) bofs = bias_fill<true>(x, g_in_b, bias_mem, 64 * kNW) + 4 * (31 - l32 + 8 * hl);

  f32x16 o[kNOB];
#pragma unroll
  for (int i = 0; i < kNOB; ++i)
#pragma unroll
    for (int r = 0; r < 16; ++r) o[i][r] = 0.f;
  float m_run = kNegInf, l_run = 0.f;
  constexpr float kStaleMax = std::is_same<Tr, BF16>::value ? 0x1p48f : 0x1p15f;

  // One key tile at LDS byte `st`, keys from k0. FIRST: the part's first tile,
  // which takes the row max before its exponentials; later ones take theirs
  // against the running max as it stands, and again with their own only when a
  // lane's sum passes what P's type and O hold (stale_softmax in prefill.hip), or
  // a row has met no finite logit yet (a bias of -inf).
  // MASK: the row group's last tile (diagonal, end of the keys).
  // NT > 1: the loads of the tile a ring ahead (group g, tile sub) go out between
  // the QK steps: all at once, the 8 waves' loads queue behind each other.
  // (Tiles past the reach, of one bias, read it all the same: a copy of the tile
  // that adds it to the exponents instead was 2-5 % slower for both.)
  auto tile = [&](uint32_t st, int k0, int g, int sub, auto first_tag, auto mask_tag) CA_INLINE {
    constexpr bool FIRST = decltype(first_tag)::value, MASK = decltype(mask_tag)::value;
    // bias reads: pair i of the lane's kBN / 4 (logits 2 i, 2 i + 1)
    constexpr int NB2 = BIAS ? 8 * kMB : 1;
    u32x2 br[NB2];
    if constexpr (BIAS) {
      const uint32_t ba = bofs + 4 * (uint32_t)bias_block(x, k0 - qw0 - 31);
      auto bread = [&](auto i) CA_INLINE {
        constexpr int p = 2 * decltype(i)::value;
        constexpr int off = 32 * (p >> 4) + 16 * ((p >> 3) & 1) + (p & 7);
        br[decltype(i)::value] = lds_read2_b32<off, off + 1>(ba);
      };
      for_const<NB2>(bread);
    }
    const uint32_t ka = st + kofs;
    u32x4 kr[kNKS][kMB];
    auto kread = [&](int ks) CA_INLINE {
      kr[ks][0] = lds_read_b128<0>(ka ^ (32 * ks));
      if constexpr (kMB == 2) kr[ks][kMB - 1] = lds_read_b128<32 * kRowB>(ka ^ (32 * ks));
    };
    constexpr int KD = 2;  // k-steps read ahead
#pragma unroll
    for (int ks = 0; ks < KD; ++ks) kread(ks);
    f32x16 s[kMB];
    if constexpr (BIAS) {
      wait_lgkm<kMB * KD>();
#pragma unroll
      for (int i = 0; i < NB2; ++i) {
        after_wait(br[i]);
        const uint32_t lo = br[i][0], hi = br[i][1];
        s[i >> 3][(2 * i) & 15] = __builtin_bit_cast(float, lo);
        s[i >> 3][(2 * i + 1) & 15] = __builtin_bit_cast(float, hi);
      }
    } else {
#pragma unroll
      for (int mb = 0; mb < kMB; ++mb)
#pragma unroll
        for (int r = 0; r < 16; ++r) s[mb][r] = 0.f;
    }
#pragma unroll
    for (int ks = 0; ks < kNKS; ++ks) {
      if (ks + KD < kNKS) kread(ks + KD);
      wait_lgkm_n(kMB * (KD < kNKS - 1 - ks ? KD : kNKS - 1 - ks));
#pragma unroll
      for (int mb = 0; mb < kMB; ++mb) {
        after_wait(kr[ks][mb]);
        s[mb] = Tr::mfma32(__builtin_bit_cast(vec8, kr[ks][mb]), qv[ks], s[mb]);
      }
      if constexpr (NT > 1) {
        constexpr int kEvery = kNKS / (2 * kPer);
        if (ks % kEvery == kEvery - 1) issue_one(g, sub, ks / kEvery);
        __builtin_amdgcn_sched_barrier(0);
      }
    }
    // the first V^T fragments land under the softmax
    constexpr int NST = kNOB * kKK, VD = 2;  // PV steps: O^T block st / kKK, k-step st % kKK
    u32x2 vr[NST][2];
    auto vread = [&](auto i) CA_INLINE {
      constexpr int st_ = decltype(i)::value, ob = st_ / kKK, kk = st_ % kKK;
      vr[st_][0] = lds_read_tr16<16 * kRowB * kk>((st + vofs1) ^ (64 * ob));
      vr[st_][1] = lds_read_tr16<16 * kRowB * kk>((st + vofs2) ^ (64 * ob));
    };
    for_const<VD>(vread);

    // a masked tile scales its logits before the mask, so that a masked one's
    // weight is 0 for scale 0 too
    vec8 pb[kKK];
    float sv[16 * kMB];
    // register i is key k0 + 8 hl + off
    const int last = (CAUSAL ? min(n_keys - 1, myq) : n_keys - 1) - k0 - 8 * hl;
#pragma unroll
    for (int i = 0; i < 16 * kMB; ++i) {
      sv[i] = s[i >> 4][i & 15];
      if (MASK) {
        const int off = 32 * (i >> 4) + 16 * ((i >> 3) & 1) + (i & 7);
        sv[i] = off > last ? kNegInf : sv[i] * a.scale_log2;
      }
    }
    auto settle_max = [&]() CA_INLINE {
      float t0_ = kNegInf, t1_ = kNegInf;
#pragma unroll
      for (int i = 0; i < 16 * kMB; i += 4) {
        t0_ = max3(t0_, sv[i], sv[i + 1]);
        t1_ = max3(t1_, sv[i + 2], sv[i + 3]);
      }
      const float t2 = __builtin_fmaxf(t0_, t1_);
      const float m_new = __builtin_fmaxf(m_run, pair32_max(MASK ? t2 : t2 * a.scale_log2));
      if (!FIRST) {
        const float alpha = m_new == kNegInf ? 1.f : fast_exp2(m_run - m_new);
#pragma unroll
        for (int i = 0; i < kNOB; ++i) o[i] *= alpha;
        l_run *= alpha;
      }
      m_run = m_new;
    };
    float sum[2];
    auto exp_all = [&]() CA_INLINE {
      const float msub = m_run == kNegInf ? 0.f : m_run;
#pragma unroll
      for (int i = 0; i < 16 * kMB; i += 2) {
        const float p0 = fast_exp2(MASK ? sv[i] - msub : __builtin_fmaf(sv[i], a.scale_log2, -msub));
        const float p1 = fast_exp2(MASK ? sv[i + 1] - msub : __builtin_fmaf(sv[i + 1], a.scale_log2, -msub));
        const vec2 pk = Tr::pack2(p0, p1);
        pb[i / 8][i % 8] = pk[0];
        pb[i / 8][i % 8 + 1] = pk[1];
        sum[(i / 2) & 1] = i < 4 ? p0 + p1 : sum[(i / 2) & 1] + (p0 + p1);
      }
    };
    if (FIRST) settle_max();
    exp_all();
    if (!FIRST &&
        __builtin_expect(wave_any(!(sum[0] + sum[1] <= kStaleMax) || (BIAS && m_run == kNegInf)), 0)) {
      settle_max();
      exp_all();
    }
    l_run += sum[0] + sum[1];

    // O^T += V^T P^T
    auto pv_step = [&](auto i) CA_INLINE {
      constexpr int st_ = decltype(i)::value;
      if constexpr (st_ + VD < NST) vread(std::integral_constant<int, st_ + VD>{});
      wait_lgkm<2 * (VD < NST - 1 - st_ ? VD : NST - 1 - st_)>();
      after_wait(vr[st_][0]);
      after_wait(vr[st_][1]);
      const u32x4 w = {vr[st_][0][0], vr[st_][0][1], vr[st_][1][0], vr[st_][1][1]};
      o[st_ / kKK] = Tr::mfma32(__builtin_bit_cast(vec8, w), pb[st_ % kKK], o[st_ / kKK]);
    };
    for_const<NST>(pv_step);
  };

  // NT == 1: a group's loads go out at its barrier; else with the tiles
  static_assert(NT == 1 || kGroups == 2, "all loads are awaited at a barrier");
  auto sync = [&](int g) CA_INLINE {
    wait_vmcnt<kLoads * (kGroups - 2)>();  // this wave's loads of group g landed
    __builtin_amdgcn_s_barrier();          // ... and every wave's; group g - 1 is read
    if (NT == 1) issue(g + kGroups - 1);
    return lds0 + (uint32_t)((g % kGroups) * kGroupB + part * 2 * kTileB);
  };
  // the part's i-th tile of this split is tile t0 + tile_of(i); its LDS bytes
  auto tile_of = [&](int i) CA_INLINE { return NT == 1 ? i * KS + part : i; };
  uint32_t st = 0;
  auto fetch = [&](int i) CA_INLINE { st = i % NT == 0 ? sync(i / NT) : st + 2 * kTileB; };
  auto step = [&](int i, auto first_tag, auto mask_tag) CA_INLINE {
    fetch(i);
    tile(st, (t0 + tile_of(i)) * kBN, i / NT + 1, i % NT, first_tag, mask_tag);
  };
  using T_ = std::true_type;
  using F_ = std::false_type;
  int i = 0;
  const int w_full = min(w_tiles, w_last);  // tiles before the masked one
  if (tile_of(0) < w_full) {
    step(0, T_{}, F_{});
#pragma clang loop unroll(disable)
    for (i = 1; tile_of(i) < w_full; ++i) step(i, F_{}, F_{});
  }
  if (w_full < w_tiles && tile_of(i) == w_full) {
    if (i == 0) step(i, T_{}, T_{});
    else step(i, F_{}, T_{});
    ++i;
  }
  for (; i < n_groups * NT; ++i) {
    fetch(i);
    if (NT > 1)
#pragma unroll
      for (int j = 0; j < 2 * kPer; ++j) issue_one(i / NT + 1, i % NT, j);
  }
  wait_vmcnt<0>();
  const float l_part = pair32_sum(l_run);
  if (hl == 0) {
    red_m[qg][part][l32] = m_run;
    red_l[qg][part][l32] = l_part;
  }
  __syncthreads();  // the ring is read: the parts' registers and the rows go there
  // Register r of 16 kNOB goes to part r / NR. Block (qg, dst, j), j counting
  // the other parts: [NR / 4][64 lanes] x 4 floats.
  auto block = [&](int dst, int j) CA_INLINE {
    return (f32x4*)lds + ((qg * KS + dst) * (KS - 1) + j) * (NR * 16) + lane;
  };
  f32x4 own[NR / 4];
#pragma unroll
  for (int dst = 0; dst < KS; ++dst) {
    f32x4 y[NR / 4];
#pragma unroll
    for (int j = 0; j < NR / 4; ++j)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int i = dst * NR + 4 * j + e;
        y[j][e] = o[i / 16][i % 16];
      }
    if (KS == 1 || dst == part) {
#pragma unroll
      for (int j = 0; j < NR / 4; ++j) own[j] = y[j];
    } else {
      f32x4* blk = block(dst, part < dst ? part : part - 1);
#pragma unroll
      for (int j = 0; j < NR / 4; ++j) blk[64 * j] = y[j];
    }
  }
  if constexpr (KS > 1) __syncthreads();
  float M = kNegInf, L = 0.f;
#pragma unroll
  for (int s = 0; s < KS; ++s) M = __builtin_fmaxf(M, red_m[qg][s][l32]);
  auto weight = [&](int s) CA_INLINE { return M == kNegInf ? 0.f : fast_exp2(red_m[qg][s][l32] - M); };
#pragma unroll
  for (int s = 0; s < KS; ++s) L += weight(s) * red_l[qg][s][l32];
  const float inv = L > 0.f ? 1.f / L : 0.f;
  const float w_own = weight(part);
#pragma unroll
  for (int j = 0; j < NR / 4; ++j) own[j] *= w_own;
#pragma unroll
  for (int p = 0; p < KS - 1; ++p) {
    const float w = weight(p < part ? p : p + 1);
    const f32x4* blk = block(part, p);
#pragma unroll
    for (int j = 0; j < NR / 4; ++j) own[j] += blk[64 * j] * w;
  }
  // register r of a 32-d block is d = 8 (r / 4) + 4 hl + r % 4
  if (a.n_split > 1) {
    const size_t pr = ((size_t)bh * rows + myq) * a.n_split + split;
    if (q_in) {
      if (part == 0 && hl == 0) a.part_lse[pr] = L > 0.f ? M + __builtin_amdgcn_logf(L) : kNegInf;
#pragma unroll
      for (int j = 0; j < NR / 4; ++j)
        *(f32x4*)(a.part_o + pr * D + 8 * (part * (NR / 4) + j) + 4 * hl) = own[j] * inv;
    }
    return;
  }
  if (a.lse && part == 0 && hl == 0 && q_in) a.lse[(size_t)bh * rows + myq] = row_lse(M, L);
  // packed into the group's rows, which its KS waves store, 16 bytes a lane
  unsigned char* orows = lds + kMeetB + qg * 32 * kRowB;
#pragma unroll
  for (int j = 0; j < NR / 4; ++j) own[j] *= inv;
  auto store_rows = [&](uint16_t* out) CA_INLINE {
#pragma unroll
    for (int j = 0; j < NR / 4; ++j) {
      const vec2 lo = Tr::pack2(own[j][0], own[j][1]), hi = Tr::pack2(own[j][2], own[j][3]);
      vec4 y;
      y[0] = lo[0]; y[1] = lo[1]; y[2] = hi[0]; y[3] = hi[1];
      const int c = part * (NR / 4) + j;  // 16-byte chunk: d = 8 c + 4 hl
      *(u32x2*)(orows + l32 * kRowB + 16 * (c ^ (l32 % Gm::kLpr)) + 8 * hl) = __builtin_bit_cast(u32x2, y);
    }
    __syncthreads();
#pragma unroll
    for (int j = 0; j < 32 * kRowB / 1024 / KS; ++j) {
      const int p = 64 * (j * KS + part) + lane, r = p / Gm::kLpr, c = p % Gm::kLpr;
      const int row = qw0 + r;
      if (row < rows)
        *(u32x4*)(out + ((size_t)bh * rows + row) * D + 8 * c) =
            *(const u32x4*)(orows + r * kRowB + 16 * (c ^ (r % Gm::kLpr)));
    }
  };
  store_rows(a.o);
  if (BIAS && a.o_low) {
    __syncthreads();
#pragma unroll
    for (int j = 0; j < NR / 4; ++j)
#pragma unroll
      for (int e = 0; e < 4; ++e) own[j][e] -= (float)Tr::pack2(own[j][e], 0.f)[0];
    store_rows(a.o_low);
  }
}

template <typename Tr, int D, class X, bool CAUSAL, int QG>
__global__ __launch_bounds__(64 * kWaves) void cross_kernel(CrossArgs a, X x) {
  extern __shared__ __attribute__((aligned(16))) unsigned char bias_mem[];
  // the splits of a tile are a launch's outermost index
  const int per_split = a.n_work;
  const int wg = (int)__builtin_amdgcn_workgroup_id_x() % per_split;
  const int split = (int)__builtin_amdgcn_workgroup_id_x() / per_split;
  const QTileWork wk = prefill_item(wg, a.n_work, a.n_qt, a.n_bh, a.order);
  const int n_pass = wk.qt1 < 0 ? 1 : 2;
#pragma clang loop unroll(disable)
  for (int pass = 0; pass < n_pass; ++pass) {
    if (pass) __syncthreads();  // every wave has stored its rows from LDS
    const auto head = x.head(pass ? wk.bh1 : wk.bh0, a.per_b);
    cross_tile<Tr, D, X, CAUSAL, QG>(a, x, bias_mem, head.bh, head.n_keys, pass ? wk.qt1 : wk.qt0, split);
  }
}

// Joins the splits' partials: one wave per row, D / 64 values a lane. Bound by
// latency: everything is loaded before the first use.
constexpr int kMaxSplits = 16;
template <typename Tr, int D>
__global__ __launch_bounds__(256) void cross_merge_kernel(const float* __restrict__ part_o,
                                                          const float* __restrict__ part_lse,
                                                          uint16_t* __restrict__ o, uint16_t* __restrict__ o_low,
                                                          float* __restrict__ lse, long long n_rows, int n_split) {
  constexpr int PER = D / 64;
  const int lane = threadIdx.x & 63;
  const long long row = (long long)blockIdx.x * 4 + (threadIdx.x >> 6);
  if (row >= n_rows) return;
  const float l = lane < n_split ? part_lse[row * n_split + lane] : kNegInf;
  float part[kMaxSplits][PER];
#pragma unroll
  for (int s = 0; s < kMaxSplits; ++s)
    if (s < n_split) {
#pragma unroll
      for (int i = 0; i < PER; ++i) part[s][i] = part_o[(row * n_split + s) * D + PER * lane + i];
    }
  float M = l;
#pragma unroll
  for (int m = kMaxSplits / 2; m >= 1; m >>= 1) M = __builtin_fmaxf(M, __shfl_xor(M, m, 64));
  M = __shfl(M, 0, 64);
  const float w = M == kNegInf ? 0.f : fast_exp2(l - M);
  float W = 0.f, acc[PER] = {};
#pragma unroll
  for (int s = 0; s < kMaxSplits; ++s)
    if (s < n_split) {
      const float ws = __shfl(w, s, 64);
      W += ws;
#pragma unroll
      for (int i = 0; i < PER; ++i) acc[i] += ws * part[s][i];
    }
  const float inv = W > 0.f ? 1.f / W : 0.f;
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    const float x = acc[i] * inv;
    Tr::store(o, row * D + PER * lane + i, x);
    if (o_low) Tr::store(o_low, row * D + PER * lane + i, x - (float)Tr::pack2(x, 0.f)[0]);
  }
  if (lse && lane == 0) lse[row] = row_lse(M, W);
}

struct CrossPlan {
  int groups = 8, n_qt = 0, order = 0, n_split = 1;
  long long grid = 0;  // without the splits
};

// Row groups per workgroup (8, 4, 2) and, where those leave the chip idle,
// splits of the key walk. Times in 0.1 us: a key step of a workgroup (64 keys of 8
// groups; 128 of 4; 128, at D = 64 256, of 2) and what a tile costs beside its
// steps, its first keys' way from HBM among it; a launch takes its busiest CU's
// rounds (of 2 groups, which fetch K and V most often, a fifth more where there is
// more than one). A split launch also writes and reads its partials and launches
// the merge. Fitted to 11 shapes x 3 group counts x 7 splits; the choice was
// within 8 % of the best there: 8 kv heads x 200 rows x 4001 keys x 128, 2 groups,
// 8 splits 17.7 us (8 groups unsplit 87, 2 unsplit 38, 2 x 16 25); 32 heads x 200 x
// 1500 x 64, 2 groups unsplit 12.3 (8: 26; 2 x 4: 19); 4 x 6000 x 6000 x 64, 4
// groups unsplit 52 (8: 87, 2: 64).
CrossPlan cross_plan(long long n_bh, int rows, int Skv, int D, bool bias, bool causal) {
  const double cus = std::max(device_cus(), 1);
  const bool d64 = D == 64;
  CrossPlan best;
  double best_cost = 0;
  for (int groups = 8; groups >= 2; groups /= 2) {
    const int keys = groups == 8 ? 64 : groups == 4 || !d64 ? 128 : 256;
    const double step = groups == 8 ? (d64 ? 9 : 12) : groups == 4 ? (d64 ? 10 : 14.5) : (d64 ? 10 : 10.5);
    const double tile = (groups == 8 ? (d64 ? 40 : 45) : groups == 4 ? 31 : 29) + (bias ? 8 : 0);
    auto rounds = [&](double wgs) {
      const double r = std::ceil(wgs / cus);
      return groups == 2 && r > 1 ? 1.2 * r : r;
    };
    CrossPlan p;
    p.groups = groups;
    p.n_qt = (rows + 32 * groups - 1) / (32 * groups);
    p.grid = prefill_grid(1, (int)n_bh, p.n_qt, causal, 1, &p.order);
    const int steps = (Skv + keys - 1) / keys;
    double cost;
    if (causal) {
      // the mean of a causal tile's steps: half the longest's and a half step
      const double mean = tile + step * (0.5 * steps + 0.5), longest = tile + step * steps;
      cost = p.order == kOrderPairs ? rounds((double)p.grid) * 2 * mean
                                    : std::max(longest, 1.1 * n_bh * p.n_qt * mean / cus);
    } else {
      cost = rounds((double)p.grid) * (tile + step * steps);
      for (int n = 2; n <= std::min(kMaxSplits, steps); ++n) {
        const double bytes = 2.0 * n_bh * rows * n * D * 4;
        const double c = rounds((double)p.grid * n) * (tile + step * ((steps + n - 1) / n)) + 45 + bytes / 4e5;
        if (c < 0.95 * cost) {
          cost = c;
          p.n_split = n;
        }
      }
    }
    if (groups == 8 || cost < 0.95 * best_cost) {
      best = p;
      best_cost = cost;
    }
  }
  return best;
}

template <typename Tr, int D, class X, bool CAUSAL>
hipError_t launch_t(CrossArgs a, const X& x, const CrossPlan& p, size_t lds, hipStream_t stream) {
  const auto kernel = p.groups == 8   ? &cross_kernel<Tr, D, X, CAUSAL, 8>
                      : p.groups == 4 ? &cross_kernel<Tr, D, X, CAUSAL, 4>
                                      : &cross_kernel<Tr, D, X, CAUSAL, 2>;
  const long long grid = p.grid * p.n_split;
  if (grid > 0x7fffffffLL / (64 * kWaves)) return hipErrorInvalidValue;
  hipLaunchKernelGGL(kernel, dim3((unsigned)grid), dim3(64 * kWaves), lds, stream, a, x);
  hipError_t e = hipGetLastError();
  if (e != hipSuccess || p.n_split <= 1) return e;
  const long long n_rows = (long long)a.n_bh * a.rows, wgs = (n_rows + 3) / 4;
  if (wgs > 0x7fffffffLL / 256) return hipErrorInvalidValue;
  hipLaunchKernelGGL((cross_merge_kernel<Tr, D>), dim3((unsigned)wgs), dim3(256), 0, stream, a.part_o, a.part_lse,
                     a.o, a.o_low, a.lse, n_rows, p.n_split);
  return hipGetLastError();
}

}  // namespace

// Whether a launch goes to decode's split walk: few enough query rows of a kv
// head to be its heads, and no LSE, which that walk does not keep. (64 x 16 heads x
// 1 x 1500 keys x 64: 41 us, 5.8 TB/s, where tiles of 64 rows, nearly all of them
// empty, pay a whole tile's products for each head.)
// float32 goes there with more rows too, where its tiles would leave most of the
// chip idle, each walking all keys. Times in us of both, fitted to 84 shapes (8
// heads x 64 rows x 4000 keys x 64: 77 in tiles, 44 here; 32 heads x 40 rows x 4000 x
// 128: 156 and 117, x 64: 82 and 92).
static bool few_rows(int dtype, const EncDecShape& s, bool bias, bool lse) {
  const long long rows = (long long)(s.Hq / s.Hkv) * s.Sq;
  if (bias || lse || (long long)s.B * s.Hq * s.Sq > 0x7fffffff) return false;
  if (rows <= 16 || rows > 256 || dtype != kDtypeF32) return rows <= 16;
  const double cus = std::max(device_cus(), 1);
  const double rounds = std::ceil((double)s.B * s.Hq * ((s.Sq + 31) / 32) / cus);
  const double tiles = 4 + 0.3e-3 * s.Skv * s.D * rounds;
  const double here = 18 + 20e-6 * s.B * s.Hkv * rows * s.Skv;
  return here < 0.9 * tiles;
}

// A launch's rows: without positions a kv head's query heads are one run of rows.
struct CrossRows {
  long long n_bh;
  int rows, per_b, ratio;
  CrossRows(const EncDecShape& s, bool bias) {
    const int G = s.Hq / s.Hkv;
    const bool packed = !bias && (long long)G * s.Sq <= 0x3fffffff;
    rows = packed ? G * s.Sq : s.Sq;
    per_b = packed ? s.Hkv : s.Hq;
    ratio = packed ? 1 : G;
    n_bh = (long long)s.B * per_b;
  }
};

size_t cross_workspace_bytes(int dtype, const EncDecShape& s, bool bias, bool causal, bool lse) {
  if (few_rows(dtype, s, bias, lse))
    return encdec_decode_bytes(dtype, s.B, s.Hq * s.Sq, s.Hkv, s.D, s.Skv);
  if (dtype == kDtypeF32) return 0;
  const CrossRows r(s, bias);
  const CrossPlan p = cross_plan(r.n_bh, r.rows, s.Skv, s.D, bias, causal);
  return p.n_split > 1 ? (size_t)r.n_bh * r.rows * p.n_split * (s.D + 1) * sizeof(float) : 0;
}

hipError_t launch_cross(int dtype, const void* q, const void* k, const void* v, void* o, float* lse,
                        const EncDecShape& s, const BiasSpec* bias, bool causal, void* ws, size_t ws_bytes,
                        hipStream_t stream) {
  if ((long long)s.B * s.Hq * s.Sq == 0) return hipSuccess;
  if (few_rows(dtype, s, bias, lse)) return launch_encdec_decode(dtype, q, k, v, o, s, nullptr, ws, ws_bytes, stream);
  if (dtype == kDtypeF32) return launch_cross_f32(q, k, v, o, lse, s, bias, causal, stream);
  CrossArgs a{(const uint16_t*)q, (const uint16_t*)k, (const uint16_t*)v, (uint16_t*)o,
              bias ? (uint16_t*)bias->o_low : nullptr, lse};
  const CrossRows r(s, bias);
  if (r.n_bh > 0x7fffffffLL) return hipErrorInvalidValue;
  a.rows = r.rows;
  a.per_b = r.per_b;
  a.ratio = r.ratio;
  a.n_bh = (int)r.n_bh;
  const float eff = bias ? bias_scale(s.scale) : s.scale;
  a.scale_log2 = __builtin_fabsf(eff) * kLog2e;
  a.q_sign = __builtin_signbit(eff) ? 0x80008000u : 0u;
  const CrossPlan p = cross_plan(r.n_bh, r.rows, s.Skv, s.D, bias, causal);
  if (p.grid > 0x7fffffffLL) return hipErrorInvalidValue;
  a.n_qt = p.n_qt;
  a.n_work = (int)p.grid;
  a.order = p.order;
  a.n_split = p.n_split;
  if (p.n_split > 1) {
    const size_t n = (size_t)r.n_bh * r.rows * p.n_split;
    if (ws_bytes < n * (s.D + 1) * sizeof(float)) return hipErrorInvalidValue;
    a.part_o = (float*)ws;
    a.part_lse = a.part_o + n * s.D;
  }
  CrossX cx;
  cx.kv_lens = s.kv_lens;
  cx.Skv = s.Skv;
  cx.B = s.B;
#define CA_CROSS_CASE(TR, DD)                                                                              \
  if (s.D == DD) {                                                                                         \
    if (!bias) return launch_t<TR, DD, CrossX, false>(a, cx, p, 0, stream);                                \
    const BiasX bx = bias_x(s, *bias, eff, 1.f / __builtin_fabsf(eff));                                         \
    const size_t lds = bias_lds_bytes(bx);                                                           \
    return causal ? launch_t<TR, DD, BiasX, true>(a, bx, p, lds, stream)                                   \
                  : launch_t<TR, DD, BiasX, false>(a, bx, p, lds, stream);                                 \
  }
  if (dtype == kDtypeBF16) {
    CA_CROSS_CASE(BF16, 64)
    CA_CROSS_CASE(BF16, 128)
  } else if (dtype == kDtypeF16) {
    CA_CROSS_CASE(F16, 64)
    CA_CROSS_CASE(F16, 128)
  }
#undef CA_CROSS_CASE
  return hipErrorInvalidValue;
}

}  // namespace ca
