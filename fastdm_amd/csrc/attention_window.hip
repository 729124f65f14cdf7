// Causal attention with a sliding window and sinks for gfx950 (bf16, head_dim 64 or 128): prompts, chunks behind a cache, single tokens.
//
//   visible   the query at place p of its sequence sees key j iff  j <= p  and  (p - j < window  or  j < sinks).  The queries of a sequence are its
//             last q_len tokens: row t is at place kv_len - q_len + t.  Rows at or past q_len, rows that see nothing,
//             and rows whose scores are all -inf, are zeros.
//   rows      the q heads that share a kv head are packed with the tokens: row r of (batch, kv head) is token r / G, head r % G, G = q_heads / kv_heads --
//             one K / V tile in LDS serves all G heads, a 32-row wave spans 32 / G tokens (less of a tile lies behind the mask), and a single
//             token's G rows are one wave's rows.
//   tiles     a block walks the key tiles its rows see, the sinks' tiles first and then the window's; tiles in between are neither read nor
//             multiplied.  A wave skips tiles none of its rows sees and masks element by element only where some row does not see some key.
//   QK^T      swapped: S^T[key][q] = K . Q^T on v_mfma_f32_32x32x16_bf16: lane (q = lane & 31, h = lane >> 5) holds 16 of each 32 keys of ITS row.
//   PV        O^T[d][q] += V^T[d][key] . P^T[key][q]: the S^T accumulator, converted pairwise to bf16, is the B operand as it is; V^T comes from the
//             row-major tile through ds_read_b64_tr_b16.  P is rounded to bf16 (at most 2^-8 of each weight, averaged over the keys; the row sums
//             are those of the unrounded weights in fp32): the matrix core's operand type.
//   softmax   one pass, running maximum and sum in fp32, exp2 domain, O and l rescaled only where a row's maximum grew by more than 2^8.
//   waves     WR waves over rows (32 each) times WK waves over the keys of a tile, merged through LDS at the end (window_plan says which).  Where the blocks
//             would not fill the chip, a block's tile list is cut into parts that run side by side and are merged by a second small launch.
//   NaN       what a row does not see does not reach it, though 0 * NaN is NaN in the matrix core: masked scores are replaced, keys past kv_len are never
//             read, values that no row of the block sees are zeroed in LDS, and a block that finds one that is not finite among those that only some
//             rows see starts over: product with the finite values, and a second product of marks for the rows that see one that is not.
//   bound     prompts: the matrix core and the softmax's VALU work behind it, which overlap across the two blocks of a CU only in part: 16384 tokens, 32/8
//             heads x 128, window 4096: 945 - 990 us (by box) = 0.97 - 1.02 PFLOP/s of visible pairs, where a large bf16 product reaches 1.19; MFMA busy
//             half of the cycles, VALU 47 %, LDS conflicts 0.  head_dim 64 (4 ragged prompts of 958 - 1531 tokens, 24 heads, window 512: 32 us): no one unit (MFMA busy
//             16 %, VALU 37 %, waiting 38 %); 960 blocks on 768 places leave a second round in which a quarter of the places work, every masked tile, half of
//             them here, passes over V in LDS between its arrival and the barrier, and the softmax takes about twice the products' cycles (its exponentials
//             alone as many).  Small grids: the chain of one block's tiles (about 1 us each for a single token).  Single tokens: HBM, 16 sequences, window 4096: 54 us = 5.0 TB/s with the merge.
//   tried     fragments read a group ahead behind scheduling fences (+3 .. 15 %, spills), a three- or four-deep ring (+1 / +12 % at head_dim 64), the
//             next tile's scores under this tile's softmax (spills at head_dim 128; +10 % at 64), s_setprio around either phase (+1 %), the row sums by
//             v_dot2 (0), 128-key tiles with eight waves (+6 %), 32-key tiles (+7 %): none of them stayed.
#include <type_traits>
#include "common.h"
#include "attn_common.h"
#include "launch.h"

namespace fdm {

// Division of 0 .. 2^31 - 1 by d, exact: i / d = (i * m) >> (32 + s) with s = ceil(log2 d) - 1 and m = ceil(2^(32 + s) / d), m < 2^32 (Granlund and Montgomery
// 1994); m = 0: d is 1.  (A division by a kernel argument is 20 instructions in a row; the ten in front of a block's first load took 0.5 us.)
struct Divider {
  uint32_t m = 0, s = 0;
  int d = 1;
  Divider() = default;
  __host__ explicit Divider(int64_t by) : d((int)by) {
    if (by <= 1) return;
    while (((int64_t)2 << s) < by) ++s;
    m = (uint32_t)((((uint64_t)1 << (32 + s)) + by - 1) / by);
  }
  __device__ __forceinline__ int operator()(int i) const { return m ? (int)(__umulhi((uint32_t)i, m) >> s) : i; }
  __device__ __forceinline__ int rest(int i) const { return i - (*this)(i) * d; }
};

struct WindowParams {
  bf16_t* o;
  const bf16_t* q;
  const bf16_t* k;
  const bf16_t* v;
  const int* q_lens;    // nullptr: sq
  const int* kv_lens;   // nullptr: sk
  int64_t q_bs, q_ts, k_bs, k_ts, v_bs, v_ts, o_bs, o_ts;
  int batch, sq, sk, kv_heads, group;
  int window, sinks;
  int n_blocks;         // row blocks of a (batch, kv head)
  int parts;            // parts a block's tile list is cut into
  int block0;           // of this launch, a multiple of 8
  int classes_log2;     // of (batch, kv head) pairs, one or more XCDs each: 1, 2, 4 or 8 classes
  Divider by_group, by_parts, by_class_pairs, by_kv_heads;
  float scale_log2e;
  float* ws_o;          // parts > 1: [batch * kv_heads * n_blocks][parts][rows of a block][D], unnormalised
  float* ws_ml;         // ... [..][..][rows][2]: maximum (exp2 domain), sum
};

// KW: keys per wave and tile; OCC: waves per SIMD that the registers have to do for.  LDS: two K / V tiles, one being worked on, one on its way
template <int D, int WR, int WK, int KW, int OCC>
__global__ void __launch_bounds__(64 * WR * WK, OCC) attn_window_kernel(const WindowParams p) {
  constexpr int NT = 64 * WR * WK, RB = 32 * WR, KT = KW * WK;
  constexpr int NKT = KW / 32;            // 32-key S^T tiles per wave and key tile
  constexpr int CPR = D / 8;              // 16-byte pieces per key
  constexpr uint32_t ROWB = D * 2;
  constexpr int TILE_BYTES = KT * D * 2;
  constexpr int LD = KT * CPR / NT;       // LDS-DMA pieces per thread and tile of K (and of V)
  constexpr int KSTEPS = D / 16, DT = D / 32;
  static_assert(KT * CPR % NT == 0 && LD >= 1);
  __shared__ __attribute__((aligned(1024))) uint8_t smem[4 * TILE_BYTES];

  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int wr = wave % WR, wk = wave / WR;
  const int lq = lane & 31, h = lane >> 5;

  // The blocks that run at one time on an XCD share its L2: a class of (batch, kv head) pairs belongs to 8 / classes XCDs (classes: the largest
  // divisor of 8 that deals the pairs out evenly), and their row blocks are taken from the last, longest lists to the first, pair by pair.
  // Against runs of consecutive row blocks per XCD: 16384 tokens, window 4096, 8 pairs 1060 -> 944 us; open window 2664 -> 1979 us.
  const int block = p.block0 + (int)blockIdx.x, xcd = block & 7, lg = p.classes_log2;
  const int it = ((block >> 3) << (3 - lg)) + (xcd >> lg);
  const int u = p.by_parts(it), part = it - u * p.parts;
  const int rb = p.n_blocks - 1 - p.by_class_pairs(u);
  const int bk = (xcd & ((1 << lg) - 1)) + (p.by_class_pairs.rest(u) << lg);
  if (rb < 0) return;
  const int unit = bk * p.n_blocks + rb;
  const int b = p.by_kv_heads(bk), kvh = bk - b * p.kv_heads;
  const int G = p.group;

  int q_len = p.sq, kv_len = p.sk;
  if (p.q_lens != nullptr) q_len = min(max(p.q_lens[b], 0), p.sq);
  if (p.kv_lens != nullptr) kv_len = min(max(p.kv_lens[b], 0), p.sk);
  q_len = __builtin_amdgcn_readfirstlane(q_len);
  kv_len = __builtin_amdgcn_readfirstlane(kv_len);
  const int first = kv_len - q_len;       // place of token 0

  // ---- this lane's row, and the places of the wave's and the block's rows
  const int n_rows = p.sq * G;
  const int row = rb * RB + wr * 32 + lq;
  const int rowc = min(row, n_rows - 1);
  const int tok = p.by_group(rowc), head = kvh * G + rowc - tok * G;
  const bool live = row < n_rows && tok < q_len;
  const int wt_lo = p.by_group(rb * RB + wr * 32), wt_hi = min(p.by_group(min(rb * RB + wr * 32 + 31, n_rows - 1)), q_len - 1);
  const int bt_lo = p.by_group(rb * RB), bt_hi = min(p.by_group(min(rb * RB + RB - 1, n_rows - 1)), q_len - 1);
  const int wp_lo = first + wt_lo, wp_hi = first + wt_hi;        // wt_lo > wt_hi: the wave has no row
  const int place = first + tok;

  // ---- the tiles the block's rows see: [0, n_sink) and [w_begin, w_end)
  int n_sink = 0, w_begin = 0, w_end = 0;
  if (bt_lo <= bt_hi && first + bt_hi >= 0) {
    const int near = max(0, first + bt_lo - p.window + 1);        // the window's first key
    const int far = min(p.sinks, near);                           // sinks in front of it
    n_sink = (far + KT - 1) / KT;
    w_begin = max(near / KT, n_sink);
    w_end = (first + bt_hi) / KT + 1;
    w_begin = min(w_begin, w_end);
  }
  const int n_list = n_sink + w_end - w_begin;
  const int i_begin = p.by_parts(part * n_list), i_end = p.by_parts((part + 1) * n_list);      // (at most 64 parts of lists of 2^24 tiles)
  auto tile_at = [&](int i) { return i < n_sink ? i : i - n_sink + w_begin; };

  const bf16_t* kbase = p.k + (int64_t)b * p.k_bs + (int64_t)kvh * D;
  const bf16_t* vbase = p.v + (int64_t)b * p.v_bs + (int64_t)kvh * D;

  // ---- Q fragments: B operand, lane holds Q[row][16 ks + 8 h .. + 8]
  i32x4 qf[KSTEPS];
  {
    const bf16_t* qp = p.q + (int64_t)b * p.q_bs + (int64_t)tok * p.q_ts + (int64_t)head * D + 8 * h;
#pragma unroll
    for (int ks = 0; ks < KSTEPS; ++ks) qf[ks] = *reinterpret_cast<const i32x4*>(qp + 16 * ks);
  }

  // ---- K / V staging by LDS-DMA: lane-linear destination, the swizzle is applied to the source.  A piece is a wave-uniform tile base plus a 32-bit
  //      lane offset that stays.  The DMA is an asm statement (it writes no register): hipcc puts s_waitcnt vmcnt(0) in front of LDS reads that
  //      follow its builtin, which is the next tile's DMA here; the waits are the two lines at the top of the loop.  Inside: one wait state between m0 and
  //      its use, five between a base that the vector unit may have written and the address.
  const uint32_t lds0 = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) uint8_t*)smem + wave * 1024;
  uint32_t kofs[LD], vofs[LD];
#pragma unroll
  for (int i = 0; i < LD; ++i) {
    const int slot = tid + i * NT, r = slot / CPR;
    kofs[i] = (uint32_t)(r * (int)p.k_ts * 2 + Swz<D>::k(r, slot % CPR) * 16);
    vofs[i] = (uint32_t)(r * (int)p.v_ts * 2 + Swz<D>::v(r, slot % CPR) * 16);
  }
  auto dma = [&](const bf16_t* base, uint32_t ofs, uint32_t lds) {
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 3\n\tglobal_load_lds_dwordx4 %1, %2" ::"s"(lds), "v"(ofs), "s"(base) : "memory");
  };
  auto stage = [&](int t, int buf) {
    const uint32_t lds = lds0 + buf * 2 * TILE_BYTES;
    const int last = kv_len - 1 - t * KT;       // >= 0: a listed tile holds a visible key
    const bf16_t* kt_ = kbase + (int64_t)t * KT * p.k_ts;
    const bf16_t* vt_ = vbase + (int64_t)t * KT * p.v_ts;
    if (last >= KT - 1) {
#pragma unroll
      for (int i = 0; i < LD; ++i) {
        dma(kt_, kofs[i], lds + i * (NT * 16));
        dma(vt_, vofs[i], lds + TILE_BYTES + i * (NT * 16));
      }
    } else {
#pragma unroll
      for (int i = 0; i < LD; ++i) {            // past the sequence: its last key again (masked)
        const int r = (tid + i * NT) / CPR, over = max(r - last, 0);
        dma(kt_, kofs[i] - (uint32_t)(over * (int)p.k_ts * 2), lds + i * (NT * 16));
        dma(vt_, vofs[i] - (uint32_t)(over * (int)p.v_ts * 2), lds + TILE_BYTES + i * (NT * 16));
      }
    }
  };

  f32x16 oacc[DT];
#pragma unroll
  for (int d = 0; d < DT; ++d)
#pragma unroll
    for (int e = 0; e < 16; ++e) oacc[d][e] = 0.f;
  float m_run = -3.0e38f, l_run = 0.f;
  constexpr float RESCALE = 8.0f;

  const int gi = lane >> 4, li = lane & 15, tq = li >> 2, tp = li & 3;
  const uint32_t kld0 = (wk * KW + lq) * ROWB + (uint32_t)Swz<D>::k(lq, h) * 16;
  uint32_t vld[DT];
#pragma unroll
  for (int d = 0; d < DT; ++d)
    vld[d] = TILE_BYTES + (wk * KW + 4 * h + tq) * ROWB + (uint32_t)Swz<D>::v(4 * h + tq, d * 4 + 2 * (gi & 1) + (tp >> 1)) * 16 + 8 * (tp & 1);

  // the n lowest bits (n < 0: none, n > 32: all)
  auto below = [](int n) -> uint32_t { return n >= 32 ? 0xffffffffu : (1u << max(n, 0)) - 1u; };

  // one key tile for this wave; base: place of its first key.  KIND 0: every row sees every key, 1: masked, 2: masked, values that are not finite apart
  auto process = [&](auto kind_c, int base, uint32_t buf) {
    constexpr int KIND = decltype(kind_c)::value;
    constexpr bool MASK = KIND != 0;
    const uint8_t* sb = smem + buf;
    f32x16 s[NKT];
#pragma unroll
    for (int n = 0; n < NKT; ++n)
#pragma unroll
      for (int e = 0; e < 16; ++e) s[n][e] = 0.f;
#pragma unroll
    for (int ks = 0; ks < KSTEPS; ++ks)
#pragma unroll
      for (int n = 0; n < NKT; ++n) {
        const i32x4 kf = *reinterpret_cast<const i32x4*>(sb + (kld0 ^ (uint32_t)(ks << 5)) + n * 32 * ROWB);
        s[n] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, kf), __builtin_bit_cast(bf16x8, qf[ks]), s[n], 0, 0, 0);
      }
    uint32_t seen[NKT];                         // MASK: bit kk of seen[n]: the row sees key base + 32 n + 4 h + kk
    if constexpr (MASK) {
#pragma unroll
      for (int n = 0; n < NKT; ++n) {
        const int at = base + n * 32 + 4 * h;
        seen[n] = (below(place - at + 1) & ~below(place - p.window - at + 1)) | (below(p.sinks - at) & below(place - at + 1));
#pragma unroll
        for (int e = 0; e < 16; ++e) {          // one v_bfe_i32 and one v_bfi_b32
          const int on = (int)(seen[n] << (31 - (e & 3) - 8 * (e >> 2))) >> 31;
          const float score = s[n][e];          // (hipcc takes the bit cast of a vector element for that of element 0)
          s[n][e] = __builtin_bit_cast(float, (__builtin_bit_cast(int, score) & on) | (~on & (int)0xff800000));
        }
      }
    }
    // row maximum: med3(a, b, +inf) is max without the canonicalisation hipcc puts in front of fmaxf
    float mx = s[0][0];
#pragma unroll
    for (int n = 0; n < NKT; ++n)
#pragma unroll
      for (int e = (n == 0 ? 1 : 0); e < 16; ++e) mx = __builtin_amdgcn_fmed3f(mx, s[n][e], __builtin_inff());
    const float mt = cross_half_max(mx) * p.scale_log2e;
    if (__any(mt > m_run + RESCALE)) {
      // row by row: a row that shares the wave with one that moves stays where it is (alpha 1), so its bits do not go by its neighbours
      const float m_new = mt > m_run + RESCALE ? mt : m_run;
      const float alpha = mt > m_run + RESCALE ? __builtin_amdgcn_exp2f(m_run - m_new) : 1.0f;
      m_run = m_new;
      l_run *= alpha;
#pragma unroll
      for (int d = 0; d < DT; ++d)
#pragma unroll
        for (int e = 0; e < 16; ++e) oacc[d][e] *= alpha;
    }
    float sum = 0.f;
    i32x4 pf[NKT][2];
#pragma unroll
    for (int n = 0; n < NKT; ++n) {
#pragma unroll
      for (int e = 0; e < 16; ++e) {
        const float w = __builtin_amdgcn_exp2f(__builtin_fmaf(s[n][e], p.scale_log2e, -m_run));
        s[n][e] = w;
        sum += w;
      }
#pragma unroll
      for (int u = 0; u < 2; ++u)
#pragma unroll
        for (int w = 0; w < 4; ++w) pf[n][u][w] = (int)pack2bf(s[n][8 * u + 2 * w], s[n][8 * u + 2 * w + 1]);
    }
    l_run += sum;
    auto vfrag = [&](int n, int u, int d) {
      const uint8_t* a = sb + vld[d] + (n * 32 + 16 * u) * ROWB;      // keys 4 h + tq, and 8 further
      return tr_pair(a, a + 8 * ROWB);
    };
#pragma unroll
    for (int n = 0; n < NKT; ++n)
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        i32x4 see;                              // KIND 2: 1.0 where the row sees the key, laid out as P
        if constexpr (KIND == 2) {
#pragma unroll
          for (int w = 0; w < 4; ++w) {
            const int k0 = 16 * u + 8 * (w >> 1) + 2 * (w & 1);
            see[w] = ((seen[n] >> k0 & 1) ? 0x3f80 : 0) | ((seen[n] >> (k0 + 1) & 1) ? 0x3f800000 : 0);
          }
        }
#pragma unroll
        for (int d = 0; d < DT; ++d) {
          i32x4 f = vfrag(n, u, d);
          if constexpr (KIND == 2) {
            i32x4 mark;
#pragma unroll
            for (int w = 0; w < 4; ++w) {
              const bool b0 = (f[w] & 0x7f80) == 0x7f80, b1 = (f[w] & 0x7f800000) == 0x7f800000;
              mark[w] = (b0 ? 0x3f80 : 0) | (b1 ? 0x3f800000 : 0);
              f[w] &= ~((b0 ? 0xffff : 0) | (b1 ? (int)0xffff0000 : 0));
            }
            f32x16 count;
#pragma unroll
            for (int e = 0; e < 16; ++e) count[e] = 0.f;
            count = __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, mark), __builtin_bit_cast(bf16x8, see), count, 0, 0, 0);
#pragma unroll
            for (int e = 0; e < 16; ++e) oacc[d][e] = count[e] > 0.f ? __builtin_nanf("") : oacc[d][e];
          }
          oacc[d] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, f), __builtin_bit_cast(bf16x8, pf[n][u]), oacc[d], 0, 0, 0);
          if constexpr (KIND == 2) __builtin_amdgcn_sched_barrier(0);
        }
      }
  };

  // ---- the list in three stretches: [sinks, the window's lower edge) masked, [mid_lo, mid_hi) seen whole by every row of the block, the diagonal masked
  //      (one loop with both bodies in it costs more registers than the kernel has)
  int mid_lo = n_sink, mid_hi = n_sink;
  if (n_list > 0) {
    const int under = first + bt_hi - p.window;                    // the last key that some row does not see below its window
    const int t_lo = under >= 0 ? under / KT + 1 : 0, t_hi = max(0, first + bt_lo + 1) / KT;
    mid_lo = min(n_sink + max(t_lo - w_begin, 0), n_list);
    mid_hi = max(min(n_sink + t_hi - w_begin, n_list), mid_lo);
  }
  const bool has_rows = wt_lo <= wt_hi;
  // a masked tile's values, each thread its own pieces: zeroes for keys that no row of the block sees; the largest magnitude of the others is kept
  u16x2 top = {0, 0};
  const int bp_lo = first + bt_lo, bp_hi = first + bt_hi;
  auto clean = [&](int base, int buf) {
    uint8_t* sv = smem + buf * 2 * TILE_BYTES + TILE_BYTES + tid * 16;
#pragma unroll
    for (int j = 0; j < LD; ++j) {
      const int key = base + (tid + j * NT) / CPR;
      i32x4* piece = reinterpret_cast<i32x4*>(sv + j * (NT * 16));
      if ((key > bp_hi) | ((key <= bp_lo - p.window) & (key >= p.sinks))) {
        *piece = i32x4{0, 0, 0, 0};
      } else {
        const i32x4 f = *piece;
#pragma unroll
        for (int w = 0; w < 4; ++w) top = __builtin_elementwise_max(top, __builtin_bit_cast(u16x2, f[w] & 0x7fff7fff));
      }
    }
  };
  int buf = 0, i = i_begin;
  auto arrive = [&](bool masked) {                      // tile i is there, tile i + 1 on its way
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");    // this wave's pieces of tile i have landed ...
    if (masked) clean(tile_at(i) * KT, buf);
    __syncthreads();                                    // ... and everybody's; the other slot has been read
    if (i + 1 < i_end) stage(tile_at(i + 1), buf ^ 1);
  };
  auto on = [&]() {
    ++i;
    buf ^= 1;
  };
  if (i_begin < i_end) stage(tile_at(i_begin), 0);
#pragma unroll
  for (int ks = 0; ks < KSTEPS; ++ks) asm volatile("" ::"v"(qf[ks]));      // (there before the loop: its waits count DMAs alone)
  for (int stretch = 0; stretch < 3; ++stretch) {
    const int to = min(stretch == 0 ? mid_lo : stretch == 1 ? mid_hi : n_list, i_end);
    if (stretch == 1) {
      for (; i < to; on()) {
        arrive(false);
        if (has_rows) process(std::integral_constant<int, 0>{}, 0, buf * 2 * TILE_BYTES);
      }
    } else {
      for (; i < to; on()) {
        arrive(true);
        const int base = tile_at(i) * KT + wk * KW;
        if (has_rows && base <= wp_hi && (base + KW > wp_lo - p.window + 1 || base < p.sinks)) process(std::integral_constant<int, 1>{}, base, buf * 2 * TILE_BYTES);
      }
    }
  }
  if (__syncthreads_or((top[0] >= 0x7f80) | (top[1] >= 0x7f80))) {      // (exponent all ones) once more from the start, with care
#pragma unroll
    for (int d = 0; d < DT; ++d)
#pragma unroll
      for (int e = 0; e < 16; ++e) oacc[d][e] = 0.f;
    m_run = -3.0e38f;
    l_run = 0.f;
    buf = 0;
    i = i_begin;
    if (i_begin < i_end) stage(tile_at(i_begin), 0);
    for (; i < i_end; on()) {
      arrive(true);
      const int base = tile_at(i) * KT + wk * KW;
      if (has_rows && base <= wp_hi && (base + KW > wp_lo - p.window + 1 || base < p.sinks)) process(std::integral_constant<int, 2>{}, base, buf * 2 * TILE_BYTES);
    }
  }

  float l_tot = l_run + __shfl_xor(l_run, 32, 64);
  if constexpr (WK > 1) {
    // ---- the key waves' shares are merged through LDS by the first of them, register by register (the same rows lie in the same lanes)
    constexpr int R4 = DT * 4;                            // f32x4 per lane
    static_assert((WK - 1) * WR * 64 * (R4 * 16 + 8) <= 4 * TILE_BYTES);
    f32x4* so = reinterpret_cast<f32x4*>(smem);
    float* sml = reinterpret_cast<float*>(smem + (WK - 1) * WR * R4 * 1024);
    __syncthreads();                                      // the last tile has been read
    if (wk > 0) {
      const int w = (wk - 1) * WR + wr;
#pragma unroll
      for (int d = 0; d < DT; ++d)
#pragma unroll
        for (int g4 = 0; g4 < 4; ++g4)
          so[(w * R4 + d * 4 + g4) * 64 + lane] = f32x4{oacc[d][4 * g4], oacc[d][4 * g4 + 1], oacc[d][4 * g4 + 2], oacc[d][4 * g4 + 3]};
      sml[w * 128 + lane] = m_run;
      sml[w * 128 + 64 + lane] = l_tot;
    }
    __syncthreads();
    if (wk > 0) return;
#pragma unroll
    for (int k2 = 1; k2 < WK; ++k2) {
      const int w = (k2 - 1) * WR + wr;
      const float m2 = sml[w * 128 + lane], m_new = fmaxf(m_run, m2);
      const float a1 = __builtin_amdgcn_exp2f(m_run - m_new), a2 = __builtin_amdgcn_exp2f(m2 - m_new);
      m_run = m_new;
      l_tot = l_tot * a1 + sml[w * 128 + 64 + lane] * a2;
#pragma unroll
      for (int d = 0; d < DT; ++d)
#pragma unroll
        for (int g4 = 0; g4 < 4; ++g4) {
          const f32x4 x = so[(w * R4 + d * 4 + g4) * 64 + lane];
#pragma unroll
          for (int c = 0; c < 4; ++c) oacc[d][4 * g4 + c] = oacc[d][4 * g4 + c] * a1 + x[c] * a2;
        }
    }
  }
  if (row >= n_rows) return;
  if (p.parts > 1) {
    const int64_t at = ((int64_t)unit * p.parts + part) * RB + wr * 32 + lq;
    float* wo = p.ws_o + at * D + 4 * h;
#pragma unroll
    for (int d = 0; d < DT; ++d)
#pragma unroll
      for (int g4 = 0; g4 < 4; ++g4)
        *reinterpret_cast<f32x4*>(wo + 32 * d + 8 * g4) = f32x4{oacc[d][4 * g4], oacc[d][4 * g4 + 1], oacc[d][4 * g4 + 2], oacc[d][4 * g4 + 3]};
    if (h == 0) {
      p.ws_ml[at * 2] = m_run;
      p.ws_ml[at * 2 + 1] = l_tot;
    }
    return;
  }
  const int keep = live && l_tot != 0.f ? -1 : 0;
  const float inv = 1.0f / l_tot;
  bf16_t* op = p.o + (int64_t)b * p.o_bs + (int64_t)tok * p.o_ts + (int64_t)head * D + 4 * h;
#pragma unroll
  for (int d = 0; d < DT; ++d)
#pragma unroll
    for (int g4 = 0; g4 < 4; ++g4) {
      i32x2 w;
      w[0] = (int)pack2bf(oacc[d][4 * g4] * inv, oacc[d][4 * g4 + 1] * inv) & keep;
      w[1] = (int)pack2bf(oacc[d][4 * g4 + 2] * inv, oacc[d][4 * g4 + 3] * inv) & keep;
      *reinterpret_cast<i32x2*>(op + 32 * d + 8 * g4) = w;
    }
}

// ---- merge of the parts: o = sum_i 2^(m_i - m) O_i / sum_i 2^(m_i - m) l_i.  D / 4 threads per row and part group; PG groups take the parts in turn (long
//      lists of parts are a chain of loads otherwise) and are joined through LDS, all in a fixed order.
template <int D, int PG>
__global__ void __launch_bounds__(256) attn_window_merge_kernel(const WindowParams p, int rb_rows) {
  constexpr int TPR = D / 4, ROWS = 256 / (TPR * PG);
  const int64_t n_rows = (int64_t)p.sq * p.group;
  const int pg = threadIdx.x / TPR % PG, lane = threadIdx.x % TPR, r_blk = threadIdx.x / (TPR * PG);
  const int64_t idx = (int64_t)blockIdx.x * ROWS + r_blk;
  const bool there = idx < n_rows * p.batch * p.kv_heads;
  const int64_t bk = there ? idx / n_rows : 0, row = there ? idx % n_rows : 0;
  const int64_t unit = bk * p.n_blocks + row / rb_rows;
  const int64_t first = unit * p.parts * rb_rows + row % rb_rows;       // part i's row: + i * rb_rows
  float m = -3.0e38f, l = 0.f;
  f32x4 acc = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
  for (int i = pg; i < p.parts; i += PG) {
    const int64_t at = first + (int64_t)i * rb_rows;
    const f32x4 x = *reinterpret_cast<const f32x4*>(p.ws_o + at * D + lane * 4);
    const float m2 = p.ws_ml[at * 2], l2 = p.ws_ml[at * 2 + 1];
    const float m_new = fmaxf(m, m2), a1 = __builtin_amdgcn_exp2f(m - m_new), a2 = __builtin_amdgcn_exp2f(m2 - m_new);
    m = m_new;
    l = l * a1 + l2 * a2;
#pragma unroll
    for (int c = 0; c < 4; ++c) acc[c] = acc[c] * a1 + x[c] * a2;
  }
  if constexpr (PG > 1) {
    __shared__ f32x4 so[256];
    __shared__ float sm[256], sl[256];
    so[threadIdx.x] = acc;
    sm[threadIdx.x] = m;
    sl[threadIdx.x] = l;
    __syncthreads();
    if (pg > 0) return;
#pragma unroll
    for (int g = 1; g < PG; ++g) {
      const int t = threadIdx.x + g * TPR;
      const f32x4 x = so[t];
      const float m_new = fmaxf(m, sm[t]), a1 = __builtin_amdgcn_exp2f(m - m_new), a2 = __builtin_amdgcn_exp2f(sm[t] - m_new);
      m = m_new;
      l = l * a1 + sl[t] * a2;
#pragma unroll
      for (int c = 0; c < 4; ++c) acc[c] = acc[c] * a1 + x[c] * a2;
    }
  }
  if (!there) return;
  const int b = (int)(bk / p.kv_heads), kvh = (int)(bk % p.kv_heads);
  const int tok = (int)(row / p.group), head = kvh * p.group + (int)(row % p.group);
  int q_len = p.sq;
  if (p.q_lens != nullptr) q_len = min(max(p.q_lens[b], 0), p.sq);
  const int keep = tok < q_len && l != 0.f ? -1 : 0;
  const float inv = 1.0f / l;
  const i32x2 w = {(int)pack2bf(acc[0] * inv, acc[1] * inv) & keep, (int)pack2bf(acc[2] * inv, acc[3] * inv) & keep};
  *reinterpret_cast<i32x2*>(p.o + (int64_t)b * p.o_bs + (int64_t)tok * p.o_ts + (int64_t)head * D + lane * 4) = w;
}

template <int D>
static int launch_merge(const WindowParams& p, int rb_rows, hipStream_t s) {
  const int64_t rows = (int64_t)p.batch * p.kv_heads * p.sq * p.group;      // (parts: fewer units than places on the chip, so one launch holds them)
  if (p.parts > 4) {
    constexpr int PG = 256 / (D / 4);
    attn_window_merge_kernel<D, PG><<<dim3((unsigned)rows), dim3(256), 0, s>>>(p, rb_rows);
  } else {
    constexpr int per = 256 / (D / 4);
    attn_window_merge_kernel<D, 1><<<dim3((unsigned)((rows + per - 1) / per)), dim3(256), 0, s>>>(p, rb_rows);
  }
  FDM_CHECK_LAUNCH();
  return FDM_OK;
}

// ---- host side: what the kernel's 32-bit numbers hold (places, rows and items; addresses are 64-bit).  Within these limits the plan's 64-bit counts are exact.
static bool window_fits(int64_t batch, int64_t sq, int64_t sk, int64_t kv_heads, int64_t group) {
  return batch <= (1 << 24) && sq <= (1 << 29) && sk <= (1 << 29) && sq * group <= (1 << 30) && batch * kv_heads <= (1 << 28);
}

// ---- which form, and into how many parts
//   0  up to 32 rows (single tokens and the like), 32-key tiles: blocks of one wave, no barrier to wait at, four (head_dim 64: eight) of them on a CU, each
//      with its own share of the list.  Four waves on a 128-key tile instead: 128 sequences of 512 keys, 32/8 heads x 128: 42 -> 59 us; one sequence,
//      window 4096: 11 -> 15 us.
//   1  the chip full of 128-row blocks: four row waves, 64-key tiles, two (head_dim 64: three) blocks on a CU whose phases drift apart, so that one's
//      softmax runs under the other's products.  64-row blocks read each tile twice as often: 16384 tokens, window 4096: 1055 -> 1593 us.
//   2  up to one 128-row block per CU: 64-row blocks of two row waves x two key waves, two of them on a CU.  Against form 3: 600 tokens, 24 heads x 64:
//      12.1 -> 9.7 us, x 128: 17.2 -> 13.5 us; 1200 tokens, 24 x 128: 26.6 -> 24.5 us.
//   3  the same with long lists (2048 keys and more, head_dim 128): 128-row blocks, four row waves x two key waves, half the reads of form 2.  Against
//      form 2: 8 sequences of 64 tokens, window 4096: 60.2 -> 53.4 us; 512-token chunks of 2, window 2048: 47.7 -> 46.0 us.
struct WindowPlan {
  int form, rb_rows, kt;
  int64_t n_blocks, units;
  int parts;
};
static WindowPlan window_plan(int64_t batch, int64_t sq, int64_t sk, int64_t kv_heads, int64_t group, int head_dim, int64_t window, int64_t sinks) {
  WindowPlan w{};
  const int64_t rows = sq * group, cus = device_cu_count();
  int64_t keys = 128 / group + 1 + window + sinks;       // that the lists of 128 rows hold at most, whatever the lengths on the device say
  if (keys > sk) keys = sk;
  w.form = rows <= 32 ? 0 : batch * kv_heads * ((rows + 127) / 128) > cus ? 1 : head_dim == 128 && keys >= 2048 ? 3 : 2;
  w.rb_rows = w.form == 0 ? 32 : w.form == 2 ? 64 : 128;
  w.kt = w.form == 0 ? 32 : w.form == 3 ? 128 : w.form == 1 || head_dim == 128 ? 64 : 128;
  w.n_blocks = (rows + w.rb_rows - 1) / w.rb_rows;
  w.units = batch * kv_heads * w.n_blocks;
  // where the blocks leave places on the chip free: parts of at least two (form 0) or four tiles; not for lists under 16 tiles, the merge is a launch of
  // its own (one token, window 128: 8.1 us in one part, 7.3 in two, but 5 us more on the host)
  const int64_t slots = cus * (w.form == 0 ? (head_dim == 128 ? 4 : 8) : w.form == 3 ? 1 : 2);
  const int64_t tiles = (keys + w.kt - 1) / w.kt;
  int64_t parts = 1;
  if (w.units < slots && tiles >= 16) {
    parts = slots / w.units;
    const int64_t most = tiles / (w.form == 0 ? 2 : 4);
    if (parts > most) parts = most;
    if (parts > 64) parts = 64;
  }
  w.parts = (int)parts;
  return w;
}

template <int D, int WR, int WK, int KW, int OCC>
static int launch_window(WindowParams p, hipStream_t s) {
  const int64_t per_class = (((int64_t)p.batch * p.kv_heads) >> p.classes_log2) * p.n_blocks * p.parts, xcds = 8 >> p.classes_log2;
  const int64_t grid = (per_class + xcds - 1) / xcds * 8;
  return launch_pieces(grid, 64 * WR * WK, [&](int64_t first, unsigned count) -> int {
    p.block0 = (int)first;
    attn_window_kernel<D, WR, WK, KW, OCC><<<dim3(count), dim3(64 * WR * WK), 0, s>>>(p);
    FDM_CHECK_LAUNCH();
    return FDM_OK;
  });
}

}  // namespace fdm

using namespace fdm;

extern "C" {

int64_t fdm_attn_window_workspace_bytes(int64_t batch, int64_t sq, int64_t sk, int q_heads, int kv_heads, int head_dim, int64_t window, int64_t sinks) {
  if (batch <= 0 || sq <= 0 || sk <= 0 || q_heads <= 0 || kv_heads <= 0 || q_heads % kv_heads || (head_dim != 64 && head_dim != 128) || window < 1 || sinks < 0) return 0;
  if (!window_fits(batch, sq, sk, kv_heads, q_heads / kv_heads)) return 0;
  const WindowPlan w = window_plan(batch, sq, sk, kv_heads, q_heads / kv_heads, head_dim, window < sk ? window : sk, sinks < sk ? sinks : sk);
  return w.parts > 1 ? w.units * w.parts * w.rb_rows * (head_dim + 2) * 4 : 0;
}

int fdm_attn_window(void* o, const void* q, const void* k, const void* v, const int32_t* q_lens, const int32_t* kv_lens, int64_t batch, int64_t sq,
                    int64_t sk, int q_heads, int kv_heads, int head_dim, int64_t q_batch_stride, int64_t q_tok_stride, int64_t k_batch_stride,
                    int64_t k_tok_stride, int64_t v_batch_stride, int64_t v_tok_stride, int64_t o_batch_stride, int64_t o_tok_stride, float scale,
                    int64_t window, int64_t sinks, void* workspace, int64_t workspace_bytes, fdm_stream_t stream) {
  (void)hipGetLastError();  // drop any stale error of an earlier, unrelated runtime call: FDM_CHECK_LAUNCH must see only ours
  if (batch < 0 || sq < 0 || sk < 0 || q_heads <= 0 || kv_heads <= 0 || q_heads % kv_heads || window < 1 || sinks < 0) return FDM_ERR_INVALID;
  if (!(scale > 0.f) || scale > 3.0e38f) return FDM_ERR_INVALID;
  if (head_dim != 64 && head_dim != 128) return FDM_ERR_UNSUPPORTED;
  if (batch == 0 || sq == 0) return FDM_OK;
  if (!o || !q || (sk > 0 && (!k || !v))) return FDM_ERR_INVALID;
  const uintptr_t at = reinterpret_cast<uintptr_t>(o) | reinterpret_cast<uintptr_t>(q) | reinterpret_cast<uintptr_t>(k) | reinterpret_cast<uintptr_t>(v);
  const int64_t strides = q_batch_stride | q_tok_stride | k_batch_stride | k_tok_stride | v_batch_stride | v_tok_stride | o_batch_stride | o_tok_stride;
  if ((at & 15) || (strides & 7) || strides < 0) return FDM_ERR_INVALID;
  if ((reinterpret_cast<uintptr_t>(q_lens) | reinterpret_cast<uintptr_t>(kv_lens)) & 3) return FDM_ERR_INVALID;
  const int64_t group = q_heads / kv_heads;
  if (k_tok_stride > (1 << 22) || v_tok_stride > (1 << 22)) return FDM_ERR_UNSUPPORTED;      // (a tile's lane offsets are 32-bit)
  if (!window_fits(batch, sq, sk, kv_heads, group)) return FDM_ERR_UNSUPPORTED;
  const int64_t win = window < sk ? window : (sk > 0 ? sk : 1), snk = sinks < sk ? sinks : sk;      // the same keys, and no overflow
  const WindowPlan w = window_plan(batch, sq, sk, kv_heads, group, head_dim, win, snk);
  const int64_t items = w.units * w.parts;
  if (items > (1 << 28)) return FDM_ERR_UNSUPPORTED;
  const int64_t need = w.parts > 1 ? w.units * w.parts * w.rb_rows * (head_dim + 2) * 4 : 0;
  if (need > 0 && (!workspace || (reinterpret_cast<uintptr_t>(workspace) & 15) || workspace_bytes < need)) return FDM_ERR_INVALID;
  WindowParams p{};
  p.o = (bf16_t*)o; p.q = (const bf16_t*)q; p.k = (const bf16_t*)k; p.v = (const bf16_t*)v; p.q_lens = q_lens; p.kv_lens = kv_lens;
  p.q_bs = q_batch_stride; p.q_ts = q_tok_stride; p.k_bs = k_batch_stride; p.k_ts = k_tok_stride; p.v_bs = v_batch_stride; p.v_ts = v_tok_stride;
  p.o_bs = o_batch_stride; p.o_ts = o_tok_stride;
  p.batch = (int)batch; p.sq = (int)sq; p.sk = (int)sk; p.kv_heads = kv_heads; p.group = (int)group;
  p.window = (int)win; p.sinks = (int)snk; p.n_blocks = (int)w.n_blocks; p.parts = w.parts;
  const int64_t pairs = batch * kv_heads;
  p.classes_log2 = pairs % 8 == 0 ? 3 : pairs % 4 == 0 ? 2 : pairs % 2 == 0 ? 1 : 0;
  p.by_group = Divider(group);
  p.by_parts = Divider(w.parts);
  p.by_class_pairs = Divider(pairs >> p.classes_log2);
  p.by_kv_heads = Divider(kv_heads);
  p.scale_log2e = scale * 1.4426950408889634f;
  p.ws_o = (float*)workspace;
  p.ws_ml = p.ws_o + w.units * w.parts * w.rb_rows * head_dim;
  hipStream_t s = to_stream(stream);
  int rc;
  if (head_dim == 128)
    rc = w.form == 0 ? launch_window<128, 1, 1, 32, 1>(p, s) : w.form == 1 ? launch_window<128, 4, 1, 64, 2>(p, s) : w.form == 2 ? launch_window<128, 2, 2, 32, 2>(p, s) : launch_window<128, 4, 2, 64, 2>(p, s);
  else
    rc = w.form == 0 ? launch_window<64, 1, 1, 32, 2>(p, s) : w.form == 1 ? launch_window<64, 4, 1, 64, 3>(p, s) : launch_window<64, 2, 2, 64, 2>(p, s);
  if (rc != FDM_OK || w.parts == 1) return rc;
  return head_dim == 128 ? launch_merge<128>(p, w.rb_rows, s) : launch_merge<64>(p, w.rb_rows, s);
}

}  // extern "C"
