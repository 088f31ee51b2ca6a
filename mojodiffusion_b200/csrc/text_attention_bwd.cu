// Backward pass of the language models' attention on tcgen05 / TMEM. Two launches of one kernel template and, for a learned parameter, a small sum:
//
//   KEYS = false (dq):     a CTA owns 128 query rows of one head and streams tiles of 64 keys:
//       X = Q K^T, Y = dO V^T;  P = exp2(x - lse), dS = P (Y - delta);  dQ += dS K
//   KEYS = true (dk, dv):  a CTA owns 128 keys of one key head and streams tiles of 64 queries of every head of the group, one head after the
//       other:  X = K Q^T, Y = V dO^T;  P^T, dS^T;  dV += P^T dO, dK += dS^T Q
//
// The sums over a group's heads stay in the accumulators, so no two CTAs add to one output and the results do not depend on their order.
// delta = rowsum(do o) is formed by the first launch for its own rows and read by the second. In rows of few keys ds is a difference of nearly equal
// terms: there the rounding of o would show (relative errors of 0.0027 in dq and dk at 20 tokens instead of 0.0024), so what it left is added. So it is
// for the gradients of parameters, which add ds or delta (the table's 0.0026 at 4 x 512 tokens, 0.0024 with it).
//
// The 128-row operands stay on chip (dq: Q and dO in TMEM, KEYS: K and V in shared memory), the 64-row ones stream through a ring and serve twice:
// K-major for the score products and MN-major for the gradient products. Heads of 128: score tiles are double buffered in TMEM, one buffer per math
// warpgroup: while one warpgroup turns its tile into bf16 P / dS (over the scores, the A operand of the gradient products), the tensor core and the
// other one work on the next. Heads of 64: one buffer, whose columns the warpgroups share, and a second CTA on the SM instead.
//
// dq's rows of Q, dO and O come by TMA, through the place of the ring, and from there into TMEM and delta: with plain loads by the thread of each
// row dq of 2 x 2048 tokens, 32 / 8 heads of 128, window 512 took 127 us instead of 103; with 4 x 512 tokens, 64 heads of 64 and a table 107 instead of 91.
//
// What bounds it: the latency of the turns between the products and the exponentials of a tile. Heads of 128, the case above: tensor pipe active 33 % of the
// cycles in dq (93 us) and 44 % in KEYS (122 us), issue slots 30 and 31 %. Heads of 64 with a table: 12 and 19 %, issue slots 46 % in both (90 and 83 us);
// there the scores of a tile are only formed when all eight math warps are done with the one before. With short windows also the starts and ends of CTAs:
// 1531 tokens, 64 / 8 heads of 64, window 128: dq 768 CTAs of four or five tiles, issue slots 34 %.
//
// Only tiles in which a pair may be visible are streamed; in those that are not visible whole, each thread makes its row's visibility bits.
// Rows of K and V that no query of the CTA sees are zeroed in shared memory before they are multiplied (0 * NaN is not 0).
//
// dtable (BIAS, first launch): dS is summed by bucket, in fp32 before it is rounded. In a block of 32 rows (a warp) x 32 keys whose distances lie
// in one bucket a thread adds its 32 values to its accumulator of that bucket. In the others, near the diagonal, it writes the running sums
// of its 32 values to shared memory: the sum over the distances of a bucket is the difference of two of them, at places that the borders and the
// row give. That is one addition per value and about ten instructions per bucket of the block (sums along diagonals by shuffles take about four
// per value). Each thread has its own accumulators; they are added in a fixed order at the end.
#include "text_attention.cuh"
#include "gemm_api.h"

#include <algorithm>
#include <string.h>

namespace mdb {

constexpr int TB_THREADS = 320;      // warps: 0 TMA, 1 MMA issue, 2-5 and 6-9 two math warpgroups
constexpr int TR = 128, TC = 64;     // resident rows, rows of a streamed tile
constexpr int RUN_LD = 36;           // floats between the running sums of two rows: 16-byte stores and the skewed reads hit all banks

struct alignas(64) TextBwdMaps {
  CUtensorMap r1, r2, c1, c2;      // dq: Q, dO, K, V; KEYS: K, V, Q, dO
  CUtensorMap o, o_low;            // dq
};

// What several CTAs add to dk and dv of the same keys, in fp32 parts [B, Hkv, blocks, count, 2, TR, DH] that the last kernel adds in order.
//   slices > 0: the first `blocks` blocks hold keys that every query may see. Their first part comes from the queries of a window, like the sums of the
//               other blocks; the rest of what they stream is shared by `slices` more CTAs each. Only rows of first keys are parts.
//   slices = 0, count > 1: few blocks for the SMs: `count` CTAs share what each of them streams.
struct TextParts {
  int blocks, slices, count;
  float* ws;
};

template <int DH, bool KEYS, bool BIAS> struct TextBwdShape {
  static constexpr bool SUMMED = BIAS && !KEYS;                            // dtable is formed
  // Heads of 64: two CTAs to an SM, each with one buffer of X and Y whose columns the two warpgroups share (with dtable where its tables leave the room,
  // as for 32 buckets of distances up to 128). Heads of 128 need all of TMEM: there two buffers, one for either warpgroup.
  static constexpr int CTAS = DH == 64 ? 2 : 1, BUFS = CTAS == 2 ? 1 : 2;
  static constexpr int TMEM = CTAS == 2 ? 256 : 512;
  static constexpr int STAGES = DH == 64 && SUMMED ? 2 : 4;
  static constexpr int TILES = (KEYS ? 2 * TR * DH * 2 : 0) + STAGES * 2 * TC * DH * 2 + 1024;
  static constexpr int SUMS = SUMMED ? 8 * 32 * RUN_LD * 4 : 0;
  static __host__ __device__ int lut_bytes(int near) { return BIAS ? TextLut::bytes(near) : 0; }
  static __host__ __device__ int bytes(int near, int buckets) {
    return TILES + SUMS + lut_bytes(near) + (SUMMED ? (buckets - 1) * 256 * 4 + buckets * 4 + (2 * near + 4) : 0);
  }
};

template <int DH, bool KEYS, bool BIAS>
__global__ void __launch_bounds__(TB_THREADS, TextBwdShape<DH, KEYS, BIAS>::CTAS)
text_bwd_kernel(const __grid_constant__ TextBwdMaps maps, const __grid_constant__ MdbTextAttnArgs a, const TextParts parts) {
  using Shape = TextBwdShape<DH, KEYS, BIAS>;
  constexpr int STAGES = Shape::STAGES, BUFS = Shape::BUFS;
  constexpr bool SUMMED = Shape::SUMMED;
  constexpr int PLACES = 3 - BUFS;       // KEYS: where a warpgroup's queries are staged in turn, each place with a barrier of its own
  constexpr int DBOX = DH / 64;
  constexpr int R_BYTES = TR * DH * 2, R_BOX = TR * 128;
  constexpr int C_BYTES = TC * DH * 2, C_BOX = TC * 128;
  constexpr uint32_t X_COL = 0, Y_COL = BUFS * TC, ACC1_COL = 2 * BUFS * TC, ACC2_COL = ACC1_COL + DH;      // X buffers | Y buffers | dQ or dK | dV
  constexpr uint32_t AQ_COL = ACC1_COL + DH, AD_COL = AQ_COL + DH / 2;                                 // dq: Q | dO, bf16 pairs

  extern __shared__ uint8_t smem_raw[];
  __shared__ uint64_t r_full, c_full[STAGES], c_empty[STAGES], xy_full[2], pds_full[2], lv_full[2][PLACES], acc_full, a_full;
  __shared__ uint32_t tmem_base_s;
  __shared__ int abort_s;
  __shared__ __align__(16) float s_lse[2][TC], s_delta[2][TC];      // negated, per staged query: of either buffer, or of either warpgroup's columns, twice

  const uint32_t raw_addr = smem_u32(smem_raw);
  uint8_t* smem = smem_raw + (((raw_addr + 1023u) & ~1023u) - raw_addr);
  uint8_t* sR1 = smem;
  uint8_t* sR2 = sR1 + R_BYTES;
  uint8_t* sC = KEYS ? sR2 + R_BYTES : smem;                              // STAGES x (C1, C2)
  const int near = BIAS ? text_near(a) : 0;
  // dq: o_low, Q, dO and O of the rows come in where the stages and the running sums will be. Without o_low the first stage is loaded with them.
  static_assert(KEYS || Shape::TILES - 1024 + Shape::SUMS >= 4 * R_BYTES);
  const int at_once = KEYS ? STAGES : a.o_low == nullptr ? 1 : 0;
  float* sums = reinterpret_cast<float*>(sC + STAGES * 2 * C_BYTES);      // SUMMED: running sums [8 warps][32 rows][RUN_LD]
  const TextLut lut(sums + Shape::SUMS / 4, near);                        // BIAS
  float* bins = reinterpret_cast<float*>(reinterpret_cast<uint8_t*>(sums) + Shape::SUMS + Shape::lut_bytes(near));      // SUMMED: [buckets - 1][256 threads]: dS of a row before its first key of the second run, the third, ... and in all
  // SUMMED: the buckets in the order of their distances ("runs"): first distance of each, and the run of the distances -near .. near
  const int run_mid = a.exact + a.n_borders, runs = 2 * run_mid + 1;
  int* run_start = reinterpret_cast<int*>(bins + (a.buckets - 1) * 256);        // [runs]
  uint8_t* run_of = reinterpret_cast<uint8_t*>(run_start + a.buckets);

  const int warp = threadIdx.x >> 5;
  const int lane = threadIdx.x & 31;
  const int batch = blockIdx.z;
  const int rep = a.H / a.Hkv;
  // the rows with the most to stream start first: late queries, early keys
  // KEYS: blocks of keys in turn with their parts, or blocks and then the slices of the first ones
  const int key_blocks = (a.Skv + TR - 1) / TR, extra = KEYS && parts.slices > 0 ? static_cast<int>(blockIdx.x) - key_blocks : -1;
  const bool shared = KEYS && parts.slices == 0 && parts.count > 1;
  const int part = extra >= 0 ? 1 + extra % parts.slices : shared ? blockIdx.x % parts.count : 0;
  const int block = !KEYS ? (BIAS ? blockIdx.x : gridDim.x - 1 - blockIdx.x) : extra >= 0 ? extra / parts.slices : shared ? blockIdx.x / parts.count : blockIdx.x;
  const int r0 = block * TR;
  const int out_rows = KEYS ? a.Skv : a.Sq;
  const TextSight sight = text_sight(a, batch);

  // streamed tiles: keys [0, ns) and [lo, hi); queries [lo, hi) of each head of the group
  TextKeys seen = {0, 0, 0};
  int ns = 0, lo = 0, hi = 0;
  if (!KEYS) {
    seen = text_keys<BIAS>(a, sight, sight.start + r0, sight.start + min(r0 + TR, a.Sq) - 1);
    ns = (seen.sinks + TC - 1) / TC;
    lo = max(seen.lo / TC, ns);
    hi = max(seen.end > seen.lo ? (seen.end + TC - 1) / TC : lo, lo);
  } else if (r0 < sight.valid) {
    int first = 0, end = a.Sq;
    if (!BIAS) {
      first = max(r0 - sight.start, 0);
      if ((parts.slices > 0 && block < parts.blocks) || r0 >= a.sinks) end = static_cast<int>(max(min(static_cast<long long>(a.Sq), static_cast<long long>(r0) + TR - 1 + a.window - sight.start), 0ll));
    }
    if (first < end) {
      lo = first / TC;
      hi = (end + TC - 1) / TC;
    }
    if (extra >= 0) {               // the queries behind the window's
      lo = max(first / TC, hi);
      hi = max((a.Sq + TC - 1) / TC, lo);
    }
  }
  const int per_head = ns + hi - lo;
  const int n_all = KEYS ? per_head * rep : per_head;
  const int share = extra >= 0 ? part - 1 : part, shares = extra >= 0 ? parts.slices : shared ? parts.count : 1;
  const int i_first = KEYS ? static_cast<int>(static_cast<long long>(n_all) * share / shares) : 0;
  const int n_c = KEYS ? static_cast<int>(static_cast<long long>(n_all) * (share + 1) / shares) - i_first : n_all;
  const auto tile_of = [&](int i) { return i < ns ? i : i - ns + lo; };
  const auto key_seen = [&](int key) {
    long long first = 0, end = a.Sq;
    if (!BIAS) {
      first = max(key - sight.start, 0);
      if (key >= a.sinks) end = min(end, static_cast<long long>(key) + a.window - sight.start);
    }
    return key < sight.valid && first < end;
  };

  // The TMA warp makes the barriers and starts loading while the others get ready: nobody else touches either before __syncthreads.
  const int kv_head0 = KEYS ? blockIdx.y * rep + i_first / max(per_head, 1) : blockIdx.y / rep;
  int load_head = kv_head0, load_tile = KEYS ? i_first % max(per_head, 1) : 0;
  const auto load_c = [&](int st) {
    uint8_t* c1 = sC + st * 2 * C_BYTES;
    if (elect_one()) {
      mbar_expect_tx(&c_full[st], 2 * C_BYTES);
      for (int d = 0; d < DBOX; ++d) {
        tma_load_4d(c1 + d * C_BOX, &maps.c1, &c_full[st], d * 64, tile_of(load_tile) * TC, load_head, batch);
        tma_load_4d(c1 + C_BYTES + d * C_BOX, &maps.c2, &c_full[st], d * 64, tile_of(load_tile) * TC, load_head, batch);
      }
    }
    __syncwarp();
    if (++load_tile == per_head && KEYS) {
      load_tile = 0;
      ++load_head;
    }
  };
  if (warp == 0) {
    if (lane == 0) {
      mbar_init(&r_full, 1);
      for (int s = 0; s < STAGES; ++s) {
        mbar_init(&c_full[s], 1);
        mbar_init(&c_empty[s], 1);
      }
      for (int s = 0; s < 2; ++s) {
        mbar_init(&xy_full[s], 1);
        mbar_init(&pds_full[s], BUFS == 1 ? 8 : 4);
        for (int p = 0; p < PLACES; ++p) mbar_init(&lv_full[s][p], BUFS == 1 ? 32 : TC);
      }
      mbar_init(&acc_full, 1);
      mbar_init(&a_full, 8);
      abort_s = 0;
      fence_mbar_init();
    }
    __syncwarp();
    if (!KEYS || n_c > 0) {
      if (elect_one()) {
        uint8_t* to = KEYS ? sR1 : sR1 + R_BYTES;
        mbar_expect_tx(&r_full, (KEYS ? 2 : 4 - at_once) * R_BYTES);
        for (int d = 0; d < DBOX; ++d) {
          tma_load_4d(to + d * R_BOX, &maps.r1, &r_full, d * 64, r0, blockIdx.y, batch);
          tma_load_4d(to + R_BYTES + d * R_BOX, &maps.r2, &r_full, d * 64, r0, blockIdx.y, batch);
          if (!KEYS) tma_load_4d(to + 2 * R_BYTES + d * R_BOX, &maps.o, &r_full, d * 64, r0, blockIdx.y, batch);
          if (!KEYS && at_once == 0) tma_load_4d(sR1 + d * R_BOX, &maps.o_low, &r_full, d * 64, r0, blockIdx.y, batch);
        }
      }
      __syncwarp();
#pragma unroll 1
      for (int i = 0; i < at_once && i < n_c; ++i) load_c(i);
    }
  } else if (warp == 1) {
    tmem_alloc(&tmem_base_s, Shape::TMEM);
    tmem_relinquish();
  }
  if (BIAS) {
    // one head's bias: with a table there are as many key heads as query heads
    lut.set(a, blockIdx.y, warp, TB_THREADS / 32);
    if (!KEYS && a.d_table != nullptr) {
      for (int i = threadIdx.x; i < (a.buckets - 1) * 256; i += TB_THREADS) bins[i] = 0.f;
      for (int i = threadIdx.x; i <= 2 * near; i += TB_THREADS) {
        const int c = text_bucket(a, i - near);
        run_of[i] = static_cast<uint8_t>(i <= near ? run_mid - c : run_mid + c - a.buckets / 2);
      }
      for (int r = threadIdx.x; r < runs; r += TB_THREADS) {
        const int c = r < run_mid ? run_mid - r : r - run_mid;                 // bucket within its direction
        const auto reach = [&](int b) { return b <= a.exact ? b : a.borders[b - a.exact - 1]; };      // its first distance
        run_start[r] = r == 0 ? -TXT_FAR : r <= run_mid ? 1 - reach(c + 1) : reach(c);
      }
    }
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem_base = tmem_base_s;

  if (warp == 0) {
    // ----------------------------- TMA producer -----------------------------
    bool ok = true;
    int i = at_once;
    for (; i < n_c; ++i) {
      const int st = i & (STAGES - 1);
      ok = !KEYS && i < STAGES ? text_wait<DH == 128>(&a_full, 0, &abort_s) : text_wait<DH == 128>(&c_empty[st], ((i / STAGES) & 1) ^ 1u, &abort_s);
      if (!ok) break;
      load_c(st);
    }
    if (!ok) {
      if (lane == 0) report_status(a.status, STATUS_TIMEOUT, 141, i);
      // the copies on the way land before the memory is given up
      for (int j = max(i - STAGES, 0) - 1; j < i; ++j) {
        const bool r = j < max(i - STAGES, 0);
        const uint64_t t0 = globaltimer_ns();
        while (!mbar_try_wait(r ? &r_full : &c_full[j & (STAGES - 1)], r ? 0 : (j / STAGES) & 1) && globaltimer_ns() - t0 < 5000000ull) {
        }
      }
    }
    __syncwarp();
  } else if (warp == 1) {
    // ----------------------------- MMA issue --------------------------------
    if (n_c > 0) {
      constexpr uint32_t idesc_xy = make_idesc(1, UMMA_BF16, UMMA_BF16, 0, 0, TR, TC);
      constexpr uint32_t idesc_acc = make_idesc(1, UMMA_BF16, UMMA_BF16, 0, 1, TR, DH);
      const uint64_t r1 = make_desc_kmajor_sw128(smem_u32(sR1)), r2 = make_desc_kmajor_sw128(smem_u32(sR2));
      const uint64_t ck = make_desc_kmajor_sw128(smem_u32(sC)), cm = make_desc_mnmajor_sw128(smem_u32(sC), C_BOX);
      const auto issue_xy = [&](int st, int buf) {
        const uint64_t c1 = ck + static_cast<uint64_t>(st * (2 * C_BYTES >> 4)), c2 = c1 + (C_BYTES >> 4);
        const uint32_t x = tmem_base + X_COL + buf * TC, y = tmem_base + Y_COL + buf * TC;
#pragma unroll
        for (int kk = 0; kk < DH / 16; ++kk)
          if (KEYS) umma_f16_ss(x, r1 + (((kk / 4) * R_BOX + (kk % 4) * 32) >> 4), c1 + (((kk / 4) * C_BOX + (kk % 4) * 32) >> 4), idesc_xy, kk != 0 ? 1u : 0u);
          else umma_f16_ts(x, tmem_base + AQ_COL + kk * 8, c1 + (((kk / 4) * C_BOX + (kk % 4) * 32) >> 4), idesc_xy, kk != 0 ? 1u : 0u);
#pragma unroll
        for (int kk = 0; kk < DH / 16; ++kk)
          if (KEYS) umma_f16_ss(y, r2 + (((kk / 4) * R_BOX + (kk % 4) * 32) >> 4), c2 + (((kk / 4) * C_BOX + (kk % 4) * 32) >> 4), idesc_xy, kk != 0 ? 1u : 0u);
          else umma_f16_ts(y, tmem_base + AD_COL + kk * 8, c2 + (((kk / 4) * C_BOX + (kk % 4) * 32) >> 4), idesc_xy, kk != 0 ? 1u : 0u);
        umma_commit(&xy_full[buf]);
      };
      const auto issue_acc = [&](int st, int buf, bool first) {
        const uint64_t c1 = cm + static_cast<uint64_t>(st * (2 * C_BYTES >> 4)), c2 = c1 + (C_BYTES >> 4);
#pragma unroll
        for (int kk = 0; kk < TC / 16; ++kk)
          umma_f16_ts(tmem_base + ACC1_COL, tmem_base + Y_COL + buf * TC + kk / 2 * 32 + kk % 2 * 8, c1 + (kk * 2048 >> 4), idesc_acc, (first && kk == 0) ? 0u : 1u);
        if (KEYS) {
#pragma unroll
          for (int kk = 0; kk < TC / 16; ++kk)
            umma_f16_ts(tmem_base + ACC2_COL, tmem_base + X_COL + buf * TC + kk / 2 * 32 + kk % 2 * 8, c2 + (kk * 2048 >> 4), idesc_acc, (first && kk == 0) ? 0u : 1u);
        }
      };
      // rows of a key tile that no query of the CTA sees
      const auto clean = [&](int i, int st) {
        if (KEYS) return;
        const int k0 = tile_of(i) * TC;
        if (k0 + TC <= seen.end && (k0 >= seen.lo || k0 + TC <= seen.sinks)) return;
        for (int r = lane; r < TC; r += 32) {
          const int j = k0 + r;
          if (j < seen.end && (j >= seen.lo || j < seen.sinks)) continue;
          for (int b = 0; b < 2 * DBOX; ++b)
            for (int c = 0; c < 8; ++c)
              *reinterpret_cast<uint4*>(sC + st * 2 * C_BYTES + b * C_BOX + r * 128 + ((c + r) & 7) * 16) = make_uint4(0, 0, 0, 0);
        }
        fence_proxy_async_smem();
        __syncwarp();
      };
      bool ok = text_wait<DH == 128>(KEYS ? &r_full : &a_full, 0, &abort_s) && text_wait<DH == 128>(&c_full[0], 0, &abort_s);
      if (ok) {
        tc_fence_after();
        clean(0, 0);
        if (elect_one()) issue_xy(0, 0);
        __syncwarp();
      }
      for (int i = 0; ok && i < n_c; ++i) {
        const int st = i & (STAGES - 1), stn = (i + 1) & (STAGES - 1);
        const bool more = i + 1 < n_c;
        if (more) {
          ok = text_wait<DH == 128>(&c_full[stn], ((i + 1) / STAGES) & 1, &abort_s);
          if (!ok) break;
          tc_fence_after();
          clean(i + 1, stn);
          if (BUFS == 2) {
            if (elect_one()) issue_xy(stn, (i + 1) & 1);
            __syncwarp();
          }
        }
        ok = text_wait<DH == 128>(&pds_full[BUFS == 2 ? i & 1 : 0], (BUFS == 2 ? i >> 1 : i) & 1, &abort_s);
        if (!ok) break;
        tc_fence_after();
        if (elect_one()) {
          issue_acc(st, BUFS == 2 ? i & 1 : 0, i == 0);
          umma_commit(&c_empty[st]);
          if (more && BUFS == 1) issue_xy(stn, 0);        // over scores that the products before have read
          if (!more) umma_commit(&acc_full);
        }
        __syncwarp();
      }
      if (!ok && lane == 0) report_status(a.status, STATUS_TIMEOUT, 151, n_c);
    }
    __syncwarp();
  } else {
    // ------------------------------- math: warpgroup g takes the tiles of buffer g, every second one
    // (with one buffer: 32 columns of every tile)
    const int g = (warp - 2) >> 2;
    const int quad = warp & 3;
    const int mt = quad * 32 + lane;  // row inside the resident tile == TMEM lane
    const int slot = g * 128 + mt;
    const uint32_t lane_addr = static_cast<uint32_t>(quad * 32) << 16;
    const int row = r0 + mt;
    const float sl2 = a.scale * TXT_LOG2E;
    bool ok = true;
    float my_nlse = -INFINITY, my_ndelta = 0.f;       // rows behind the last query: probabilities of zero
    if (!KEYS) {
      // Q (warpgroup 0) and dO (1) become A operands in TMEM: with 64 columns of B, A from shared memory would cost the score products 48 cycles for
      // every 32. On the way warpgroup 1 forms delta.
      const long long at = (static_cast<long long>(batch) * a.H + blockIdx.y) * a.Sq + row;
      if (row < a.Sq) my_nlse = -a.lse[at];
      ok = text_wait<DH == 128>(&r_full, 0, &abort_s);
      const uint8_t* mine = sR1 + (1 + g) * R_BYTES + mt * 128;
      float2 sum = make_float2(0.f, 0.f);
#pragma unroll 1
      for (int c = 0; c < DH / 64; ++c, mine += R_BOX) {
        uint32_t r[32];
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const uint4 u = *reinterpret_cast<const uint4*>(mine + ((e ^ (mt & 7)) << 4));
          r[4 * e] = u.x;
          r[4 * e + 1] = u.y;
          r[4 * e + 2] = u.z;
          r[4 * e + 3] = u.w;
        }
        if (g == 1) {
#pragma unroll 1
          for (int from = R_BYTES; from >= (at_once == 0 ? -2 : 1) * R_BYTES; from -= 3 * R_BYTES) {      // O, then what its rounding left
#pragma unroll
            for (int e = 0; e < 8; ++e) {
              const uint4 w = *reinterpret_cast<const uint4*>(mine + from + ((e ^ (mt & 7)) << 4));
              sum = ffma2(unpack_bf16x2(r[4 * e]), unpack_bf16x2(w.x), sum);
              sum = ffma2(unpack_bf16x2(r[4 * e + 1]), unpack_bf16x2(w.y), sum);
              sum = ffma2(unpack_bf16x2(r[4 * e + 2]), unpack_bf16x2(w.z), sum);
              sum = ffma2(unpack_bf16x2(r[4 * e + 3]), unpack_bf16x2(w.w), sum);
            }
          }
        }
        tmem_st_32x32b_x32(tmem_base + lane_addr + (g == 0 ? AQ_COL : AD_COL) + c * 32, r);
      }
      tmem_wait_st();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&a_full);
      float* deltas = &s_delta[0][0];          // [128]
      if (g == 1) {
        deltas[mt] = sum.x + sum.y;
        if (row < a.Sq) a.delta[at] = sum.x + sum.y;
      }
      asm volatile("bar.sync 1, 256;" ::: "memory");
      my_ndelta = -deltas[mt];
    }
    // KEYS: thread mt < 64 stages the negated lse and delta of query mt of the warpgroup's tile, loaded one of its tiles ahead
    float next_nlse = -INFINITY, next_ndelta = 0.f;
    constexpr int STAGERS = BUFS == 1 ? 32 : TC;          // threads of a warpgroup that stage, and queries that they stage
    int f_head = kv_head0, f_tile = KEYS ? i_first % max(per_head, 1) : 0;
    const auto fetch = [&](int ahead) {
      f_tile += ahead;
      while (f_tile >= per_head) {
        f_tile -= per_head;
        ++f_head;
      }
      const int q = (lo + f_tile) * TC + (BUFS == 1 ? g * 32 : 0) + mt;
      const bool in = q < a.Sq && f_head < (static_cast<int>(blockIdx.y) + 1) * rep;
      const long long at = (static_cast<long long>(batch) * a.H + f_head) * a.Sq + q;
      next_nlse = in ? -a.lse[at] : -INFINITY;
      next_ndelta = in ? -a.delta[at] : 0.f;
    };
    const int i_begin = BUFS == 2 ? g : 0;
    const bool stager = mt < STAGERS;                    // the same in a whole warp
    if (KEYS && stager && i_begin < n_c) fetch(i_begin);
    float sum_all = 0.f;      // SUMMED: dS of this row and warpgroup so far, which ends before key sum_end
    int sum_end = 0;
    int in_head = (KEYS ? i_first % max(per_head, 1) : 0) + i_begin;
    const uint32_t xa = tmem_base + lane_addr + X_COL + (BUFS == 2 ? g * TC : 0);
    const uint32_t ya = tmem_base + lane_addr + Y_COL + (BUFS == 2 ? g * TC : 0);
    for (int i = i_begin; i < n_c; i += BUFS) {
      const uint32_t par = (BUFS == 2 ? i >> 1 : i) & 1;
      const int place = i & (PLACES - 1), half = place * 32;      // where this tile's queries are staged
      uint64_t* staged = &lv_full[g][place];
      if (KEYS) {
        while (in_head >= per_head) in_head -= per_head;
        // Two buffers: the place was last read for tile i - 2, and the warpgroup's four warps have all arrived on pds_full[g] for it. One buffer: also for
        // tile i - 2, and the scores of tile i - 1, which this warp has seen, were only formed after all warps had arrived for it. By then
        // all warps have also left their wait for the queries of tile i - 2, the place's barrier's last phase. (A barrier for both places would
        // not do: a warp may still wait for tile i - 1's phase, and could not tell it from the one after tile i's, which has its parity.)
        bool lv_ok = true;
        if (stager) {
          if (BUFS == 2 && i >= 2) lv_ok = mbar_wait(&pds_full[g], par ^ 1u, &abort_s);
          s_lse[g][half + mt] = next_nlse;
          s_delta[g][half + mt] = next_ndelta;
          mbar_arrive(staged);
        }
        if (stager && i + BUFS < n_c) fetch(BUFS);
        ok = text_wait<DH == 128>(staged, (i >> 1) & 1, &abort_s);
        ok = __all_sync(0xffffffffu, ok && lv_ok);
        if (!ok) break;
      }
      const int c0 = tile_of(in_head) * TC;          // first key (dq) or query (KEYS) of the tile
      ok = text_wait<DH == 128>(&xy_full[BUFS == 2 ? g : 0], par, &abort_s);
      if (!ok) break;
      tc_fence_after();
      constexpr int NC = BUFS;                       // pieces of 32 columns of a thread: all of the tile's, or one
      const int piece0 = BUFS == 1 ? g : 0;
      uint32_t xr[NC][32], yr[NC][32];
      float run[NC][32];                             // BIAS dq: dS
#pragma unroll
      for (int c = 0; c < NC; ++c) {
        tmem_ld_32x32b_x32(xa + (piece0 + c) * 32, xr[c]);
        tmem_ld_32x32b_x32(ya + (piece0 + c) * 32, yr[c]);
      }
      tmem_wait_ld();
      bool whole;       // every pair of the tile is visible, or its row or query lies behind the last one and has a probability of zero anyway
      if (BIAS) whole = KEYS ? r0 + TR <= sight.valid : c0 + TC <= sight.valid;
      else if (KEYS) whole = r0 + TR <= sight.valid && r0 + TR - 1 <= sight.start + c0 && (sight.start + c0 + TC - 1 - a.window < r0 || r0 + TR <= a.sinks);
      else whole = c0 + TC <= sight.valid && c0 + TC - 1 <= sight.start + r0 && (sight.start + r0 + TR - 1 - a.window < c0 || c0 + TC <= a.sinks);
#pragma unroll
      for (int c = 0; c < NC; ++c) {
        const int b0 = c0 + (piece0 + c) * 32;
        uint32_t see = 0xffffffffu;
        if (!whole) {
          if (BIAS) see = KEYS ? (row < sight.valid ? see : 0u) : bits_below(sight.valid - b0);
          else if (KEYS) see = row < sight.valid ? ~bits_below(row - sight.start - b0) & (row < a.sinks ? see : bits_below(row + a.window - sight.start - b0)) : 0u;
          else see = text_mask(a, sight.valid, sight.start + row, b0);
        }
        // BIAS: distances of the warp's 32 x 32 block lie in d0 - 31 .. d0 + 31
        const int d0 = KEYS ? r0 + quad * 32 - b0 : b0 - (r0 + quad * 32);
        const bool uniform = BIAS && (d0 - 31 >= near || d0 + 31 <= -near);
        float one_bias = 0.f;
        const float* b = nullptr;
        if (BIAS) {
          // four neighbours in one load: distances grow along the keys, and fall along the queries
          if (uniform) one_bias = d0 > 0 ? lut.behind() : lut.before();
          else b = lut.from(KEYS ? row - b0 - 3 : b0 - row);
        }
        uint32_t pk[16], dk[16];
        const float2 sl2_2 = make_float2(sl2, sl2);
#pragma unroll
        for (int e = 0; e < 32; e += 4) {
          float nl[4], nd[4];
          if (KEYS) {
            const float4 u = *reinterpret_cast<const float4*>(&s_lse[g][half + c * 32 + e]), w = *reinterpret_cast<const float4*>(&s_delta[g][half + c * 32 + e]);
            nl[0] = u.x; nl[1] = u.y; nl[2] = u.z; nl[3] = u.w;
            nd[0] = w.x; nd[1] = w.y; nd[2] = w.z; nd[3] = w.w;
          } else {
#pragma unroll
            for (int m = 0; m < 4; ++m) {
              nl[m] = my_nlse;
              nd[m] = my_ndelta;
            }
          }
          if (BIAS) {
            float4 u = make_float4(one_bias, one_bias, one_bias, one_bias);
            if (!uniform) u = *reinterpret_cast<const float4*>(b + (KEYS ? -e : e));
            nl[0] += KEYS ? u.w : u.x;
            nl[1] += KEYS ? u.z : u.y;
            nl[2] += KEYS ? u.y : u.z;
            nl[3] += KEYS ? u.x : u.w;
          }
          const float2 x01 = ffma2(make_float2(__uint_as_float(xr[c][e]), __uint_as_float(xr[c][e + 1])), sl2_2, make_float2(nl[0], nl[1]));
          const float2 x23 = ffma2(make_float2(__uint_as_float(xr[c][e + 2]), __uint_as_float(xr[c][e + 3])), sl2_2, make_float2(nl[2], nl[3]));
          float2 p01 = make_float2(ex2_approx(x01.x), ex2_approx(x01.y)), p23 = make_float2(ex2_approx(x23.x), ex2_approx(x23.y));
          if (!whole) {
            if (!(see >> e & 1u)) p01.x = 0.f;
            if (!(see >> (e + 1) & 1u)) p01.y = 0.f;
            if (!(see >> (e + 2) & 1u)) p23.x = 0.f;
            if (!(see >> (e + 3) & 1u)) p23.y = 0.f;
          }
          const float2 d01 = fmul2(p01, fadd2(make_float2(__uint_as_float(yr[c][e]), __uint_as_float(yr[c][e + 1])), make_float2(nd[0], nd[1])));
          const float2 d23 = fmul2(p23, fadd2(make_float2(__uint_as_float(yr[c][e + 2]), __uint_as_float(yr[c][e + 3])), make_float2(nd[2], nd[3])));
          pk[e >> 1] = pack_bf16x2(p01.x, p01.y);
          pk[(e >> 1) + 1] = pack_bf16x2(p23.x, p23.y);
          dk[e >> 1] = pack_bf16x2(d01.x, d01.y);
          dk[(e >> 1) + 1] = pack_bf16x2(d23.x, d23.y);
          if (BIAS && !KEYS) {
            run[c][e] = d01.x;
            run[c][e + 1] = d01.y;
            run[c][e + 2] = d23.x;
            run[c][e + 3] = d23.y;
          }
        }
        if (KEYS) tmem_st_32x32b_x16(xa + (piece0 + c) * 32, pk);      // over scores of this piece: they are in registers by now
        tmem_st_32x32b_x16(ya + (piece0 + c) * 32, dk);
      }
      tmem_wait_st();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&pds_full[BUFS == 2 ? g : 0]);
      if (SUMMED && a.d_table != nullptr) {
        // with the tile's products under way
#pragma unroll
        for (int c = 0; c < NC; ++c) {
          const int b0 = c0 + (piece0 + c) * 32, d0 = b0 - (r0 + quad * 32);
          const int r_lo = run_of[min(max(sum_end - (r0 + quad * 32) - 32 + near, 0), 2 * near)], r_hi = run_of[min(max(d0 + 31 + near, 0), 2 * near)];
          // running sums of four pieces of eight, then of the whole
#pragma unroll
          for (int e = 1; e < 8; ++e)
#pragma unroll
            for (int m = 0; m < 32; m += 8) run[c][m + e] += run[c][m + e - 1];
#pragma unroll
          for (int m = 8; m < 32; m += 8) {
            const float base = run[c][m - 1];
            if (r_lo == r_hi) {
              run[c][m + 7] += base;
            } else {
#pragma unroll
              for (int e = 0; e < 8; ++e) run[c][m + e] += base;
            }
          }
          if (r_lo != r_hi) {
            float* mine = sums + ((warp - 2) * 32 + lane) * RUN_LD;
#pragma unroll
            for (int e = 0; e < 32; e += 4) *reinterpret_cast<float4*>(mine + e) = make_float4(run[c][e], run[c][e + 1], run[c][e + 2], run[c][e + 3]);
            // Bucket r + 1 of this row begins at key `at`: what came before it. Where that key lies in a tile of the other warpgroup, the sum so far.
#pragma unroll 4
            for (int r = r_lo; r < r_hi; ++r) {
              const int at = run_start[r + 1] + row;
              const float upto = at > b0 ? mine[min(at - b0, 32) - 1] : 0.f;
              if (at >= sum_end && at < b0 + 32) bins[r * 256 + slot] = sum_all + upto;
            }
          }
          sum_all += run[c][31];
          sum_end = b0 + 32;
        }
      }
      in_head += BUFS;
    }
    if (ok && n_c > 0) ok = text_wait<DH == 128>(&acc_full, 0, &abort_s);
    if (!ok && lane == 0) report_status(a.status, STATUS_TIMEOUT, 161, n_c);
    if (ok) {
      // dq: each warpgroup stores half of the columns; KEYS: warpgroup 0 dk, warpgroup 1 dv
      tc_fence_after();
      bool some = n_c > 0;
      if (KEYS) {
        some = some && key_seen(row);      // a key that no query sees may hold anything, and its gradient is zero
      }
      const bool second = KEYS && g == 1;
      const long long* st = !KEYS ? a.dq_strides : second ? a.dv_strides : a.dk_strides;
      // 32 columns at a time through the tiles' memory, which no product reads any more, so that a store covers 64 bytes of eight rows: dk and dv of
      // relative attention with 4 x 512 tokens and 64 heads of 64 columns take 86.5 us so, 93.7 with a row stored by each thread. The loop stays a loop: it runs once.
      uint8_t* stage = sR1 + (warp - 2) * 4096;
      const int line = r0 + quad * 32 + (lane >> 2);
      __nv_bfloat16* out = static_cast<__nv_bfloat16*>(!KEYS ? a.dq : second ? a.dv : a.dk) + batch * st[0] + line * st[1] + blockIdx.y * st[2] + (lane & 3) * 8;
      const uint32_t acc = tmem_base + lane_addr + (second ? ACC2_COL : ACC1_COL);
      const float f = second ? 1.f : a.scale;
      const auto leaves_as_part = [&](int row_) { return shared || (KEYS && parts.slices > 0 && block < parts.blocks && row_ < a.sinks); };
      const bool as_part = leaves_as_part(row);
      float* whole = as_part ? parts.ws + ((((static_cast<long long>(batch) * a.Hkv + blockIdx.y) * parts.blocks + block) * parts.count + part) * 2 + g) * (TR * DH) + mt * DH : nullptr;
      constexpr int CHUNKS = KEYS ? DH / 32 : DH / 64;
      const int first = KEYS ? 0 : g * CHUNKS;
#pragma unroll 1
      for (int c = first; c < first + CHUNKS; ++c) {
        uint32_t r[32];
        if (n_c > 0) {
          tmem_ld_32x32b_x32(acc + c * 32, r);
          tmem_wait_ld();
        }
#pragma unroll
        for (int e = 0; e < 32; ++e)
          if (!some) r[e] = 0u;
        if (as_part) {
#pragma unroll
          for (int e = 0; e < 32; e += 4) *reinterpret_cast<uint4*>(whole + c * 32 + e) = make_uint4(r[e], r[e + 1], r[e + 2], r[e + 3]);
        }
        __syncwarp();
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          uint4 w;
          w.x = pack_bf16x2(__uint_as_float(r[8 * e + 0]) * f, __uint_as_float(r[8 * e + 1]) * f);
          w.y = pack_bf16x2(__uint_as_float(r[8 * e + 2]) * f, __uint_as_float(r[8 * e + 3]) * f);
          w.z = pack_bf16x2(__uint_as_float(r[8 * e + 4]) * f, __uint_as_float(r[8 * e + 5]) * f);
          w.w = pack_bf16x2(__uint_as_float(r[8 * e + 6]) * f, __uint_as_float(r[8 * e + 7]) * f);
          *reinterpret_cast<uint4*>(stage + lane * 64 + ((e ^ (lane >> 1 & 3)) << 4)) = w;
        }
        __syncwarp();
#pragma unroll
        for (int n = 0; n < 4; ++n) {
          const int to = line + n * 8, rl = (lane >> 2) + n * 8;
          if (to < out_rows && extra < 0 && !leaves_as_part(to))
            *reinterpret_cast<uint4*>(out + n * 8 * st[1] + c * 32) = *reinterpret_cast<const uint4*>(stage + rl * 64 + (((lane & 3) ^ (rl >> 1 & 3)) << 4));
        }
      }
    }
    if (SUMMED && a.d_table != nullptr) {
      // runs that begin behind the last key, and the end of the last one
      for (int r = 1; r < runs; ++r)
        if (run_start[r] + row >= sum_end) bins[(r - 1) * 256 + slot] = sum_all;
      bins[(runs - 1) * 256 + slot] = sum_all;
      asm volatile("bar.sync 1, 256;" ::: "memory");
      float* part = a.ws + ((static_cast<long long>(batch) * a.H + blockIdx.y) * gridDim.x + blockIdx.x) * a.buckets;
      for (int c = warp - 2; c < a.buckets; c += 8) {
        const int side = c < a.buckets / 2 ? c : c - a.buckets / 2, r = c < a.buckets / 2 ? run_mid - c : run_mid + side;
        float s = 0.f;
        if (side <= run_mid && (c < a.buckets / 2 || side > 0)) {
#pragma unroll
          for (int m = 0; m < 256; m += 32) s += bins[r * 256 + m + lane] - (r > 0 ? bins[(r - 1) * 256 + m + lane] : 0.f);
        }
#pragma unroll
        for (int m = 16; m > 0; m >>= 1) s += __shfl_xor_sync(0xffffffffu, s, m);
        if (lane == 0) part[c] = s;
      }
    }
  }

  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem_base, Shape::TMEM);
  }
}

// What is left, in one launch: blocks [0, adders) add the parts of dk and dv, 32 rows of a key head of a sequence each; the others form the gradient of
// one head's sink logit, -sum of exp2(sink - lse) delta, or of its column of the table, from the sums of all row blocks and sequences. All in a fixed order.
__global__ void __launch_bounds__(256)
text_finish_kernel(const __grid_constant__ MdbTextAttnArgs a, const TextParts parts, const int part_rows, const int adders, const int row_blocks) {
  __shared__ float sums[256];
  if (static_cast<int>(blockIdx.x) < adders) {
    const int groups = a.Dh / 8, lines = (part_rows + 31) / 32;
    const int line = blockIdx.x % lines, g = blockIdx.x / lines % a.Hkv, batch = blockIdx.x / lines / a.Hkv;
    for (int e = threadIdx.x; e < 32 * 2 * groups; e += 256) {
      const int c = e % groups, m = e / groups % 2, key = line * 32 + e / groups / 2;
      if (key >= part_rows) continue;
      const float* at = parts.ws + ((((static_cast<long long>(batch) * a.Hkv + g) * parts.blocks + key / TR) * parts.count) * 2 + m) * (TR * a.Dh) + key % TR * a.Dh + c * 8;
      float s[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
      for (int p = 0; p < parts.count; ++p) {
        const float4 u = *reinterpret_cast<const float4*>(at + static_cast<long long>(p) * 2 * TR * a.Dh), v = *reinterpret_cast<const float4*>(at + static_cast<long long>(p) * 2 * TR * a.Dh + 4);
        s[0] += u.x; s[1] += u.y; s[2] += u.z; s[3] += u.w;
        s[4] += v.x; s[5] += v.y; s[6] += v.z; s[7] += v.w;
      }
      const float x = m == 0 ? a.scale : 1.f;
      const long long* st = m == 0 ? a.dk_strides : a.dv_strides;
      *reinterpret_cast<uint4*>(static_cast<__nv_bfloat16*>(m == 0 ? a.dk : a.dv) + batch * st[0] + key * st[1] + g * st[2] + c * 8) =
          make_uint4(pack_bf16x2(s[0] * x, s[1] * x), pack_bf16x2(s[2] * x, s[3] * x), pack_bf16x2(s[4] * x, s[5] * x), pack_bf16x2(s[6] * x, s[7] * x));
    }
    return;
  }
  const int h = blockIdx.x - adders, t = threadIdx.x;
  const auto store = [&](void* to, long long at, float v) {
    if (a.param_f32) static_cast<float*>(to)[at] = v;
    else static_cast<__nv_bfloat16*>(to)[at] = __float2bfloat16_rn(v);
  };
  float s = 0.f;
  if (a.d_table != nullptr) {
    const int c = t % a.buckets, group = t / a.buckets, groups = 256 / a.buckets;
    if (group < groups)
      for (int r = group; r < a.B * row_blocks; r += groups) s += a.ws[((static_cast<long long>(r / row_blocks) * a.H + h) * row_blocks + r % row_blocks) * a.buckets + c];
    sums[t] = s;
    __syncthreads();
    if (t >= a.buckets) return;
    for (int n = 1; n < groups; ++n) s += sums[n * a.buckets + c];
    store(a.d_table, static_cast<long long>(c) * a.H + h, s);
    return;
  }
  const float sink = TXT_LOG2E * text_param(a.sink_logits, a.param_f32, h);
  for (int b = 0; b < a.B; ++b) {
    const long long at = (static_cast<long long>(b) * a.H + h) * a.Sq;
#pragma unroll 4
    for (int i = t; i < a.Sq; i += 256) s += exp2f(sink - a.lse[at + i]) * a.delta[at + i];
  }
  sums[t] = s;
  __syncthreads();
  for (int n = 128; n > 0; n >>= 1) {
    if (t < n) sums[t] += sums[t + n];
    __syncthreads();
  }
  if (t == 0) store(a.d_sink, h, -sums[0]);
}

static int bwd_map(CUtensorMap* m, const void* ptr, int B, int S, int H, int Dh, const long long* strides, int rows) {
  int64_t ext[4] = {Dh, S, H, B};
  int64_t str[4] = {2, strides[1] * 2, strides[2] * 2, strides[0] * 2};
  int box[4] = {64, rows, 1, 1};
  return mdb_make_tmap(m, ptr, 2, 4, ext, str, box, 1);
}

// The start and end of a CTA take as long as about four tiles of 64 queries: slices of sixteen (2 x 2048 x 32 / 8 x 128, window 512, 4 first keys: dk and dv
// without slices 215 us, with them 132), and parts of eight at least where few blocks leave SMs idle.
// The slices of all first blocks are four CTAs per place on the SMs at most, and none where those blocks are as many by themselves: parts of 64 or 128 KB
// each, so that the workspace stays below 160 MB however many first keys there are.
static TextParts text_parts(const MdbTextAttnArgs& a) {
  TextParts p = {0, 0, 1, nullptr};
  const long long rep = a.H / a.Hkv, blocks = (a.Skv + TR - 1) / TR, groups = static_cast<long long>(a.Hkv) * a.B;
  const long long slots = (a.Dh == 64 ? 2 : 1) * device_sm_count();
  const bool windowed = a.table == nullptr && a.sinks < a.Skv;                 // with as many first keys as keys there is no window
  const long long reach = windowed ? std::min<long long>(a.Sq, static_cast<long long>(a.window) + TR) : a.Sq;      // queries of a block of keys, at most
  const long long behind = a.Sq - reach;                                       // queries that only the first keys are streamed for
  if (windowed && a.sinks > 0 && behind >= 4 * TC) {
    const long long first = (a.sinks + TR - 1) / TR;
    p.slices = static_cast<int>(std::min({(behind / TC * rep + 15) / 16, 4 * slots / (first * groups), 64ll}));
    if (p.slices > 0) {
      p.blocks = static_cast<int>(first);
      p.count = 1 + p.slices;
      return p;
    }
  }
  const long long tiles = rep * ((reach + TC - 1) / TC);
  p.count = static_cast<int>(std::max<long long>(1, std::min({slots / (blocks * groups), tiles / 8, 8ll})));
  if (p.count > 1) p.blocks = static_cast<int>(blocks);
  return p;
}
static long long part_floats(const MdbTextAttnArgs& a, const TextParts& p) {
  return static_cast<long long>(a.B) * a.Hkv * p.blocks * p.count * 2 * TR * a.Dh;
}

template <int DH, bool KEYS, bool BIAS>
static int launch_text_bwd(const TextBwdMaps& maps, const MdbTextAttnArgs& a, const TextParts& parts, cudaStream_t st) {
  using Shape = TextBwdShape<DH, KEYS, BIAS>;
  constexpr int MOST = 225 * 1024;                 // beside what the kernel declares itself
  const int smem = BIAS ? Shape::bytes(text_near(a), a.buckets) : Shape::bytes(0, 0);
  if (smem > MOST) return -6;
  auto kern = text_bwd_kernel<DH, KEYS, BIAS>;
  static bool ready[TXT_DEVICES];
  if (int r = allow_smem(kern, MOST, ready)) return r;
  int blocks = ((KEYS ? a.Skv : a.Sq) + TR - 1) / TR;
  if (KEYS) blocks = parts.slices > 0 ? blocks + parts.blocks * parts.slices : blocks * parts.count;
  kern<<<dim3(blocks, KEYS ? a.Hkv : a.H, a.B), TB_THREADS, smem, st>>>(maps, a, parts);
  return static_cast<int>(cudaGetLastError());
}

template <int DH>
static int text_backward(const MdbTextAttnArgs& a, const TextParts& parts, cudaStream_t st) {
  TextBwdMaps maps;
  memset(&maps, 0, sizeof(maps));
  int r;
  if ((r = bwd_map(&maps.c1, a.k, a.B, a.Skv, a.Hkv, DH, a.k_strides, TC))) return 1200 + r;
  if ((r = bwd_map(&maps.c2, a.v, a.B, a.Skv, a.Hkv, DH, a.v_strides, TC))) return 1300 + r;
  if ((r = bwd_map(&maps.r1, a.q, a.B, a.Sq, a.H, DH, a.q_strides, TR))) return 1400 + r;
  if ((r = bwd_map(&maps.r2, a.dout, a.B, a.Sq, a.H, DH, a.do_strides, TR))) return 1500 + r;
  if ((r = bwd_map(&maps.o, a.o, a.B, a.Sq, a.H, DH, a.o_strides, TR))) return 1600 + r;
  if (a.o_low != nullptr && (r = bwd_map(&maps.o_low, a.o_low, a.B, a.Sq, a.H, DH, a.o_strides, TR))) return 1700 + r;
  if ((r = a.table != nullptr ? launch_text_bwd<DH, false, true>(maps, a, parts, st) : launch_text_bwd<DH, false, false>(maps, a, parts, st))) return r;
  if ((r = bwd_map(&maps.r1, a.k, a.B, a.Skv, a.Hkv, DH, a.k_strides, TR))) return 2000 + r;
  if ((r = bwd_map(&maps.r2, a.v, a.B, a.Skv, a.Hkv, DH, a.v_strides, TR))) return 2100 + r;
  if ((r = bwd_map(&maps.c1, a.q, a.B, a.Sq, a.H, DH, a.q_strides, TC))) return 2200 + r;
  if ((r = bwd_map(&maps.c2, a.dout, a.B, a.Sq, a.H, DH, a.do_strides, TC))) return 2300 + r;
  return a.table != nullptr ? launch_text_bwd<DH, true, true>(maps, a, parts, st) : launch_text_bwd<DH, true, false>(maps, a, parts, st);
}

// sums of the table's gradient by row block, rounded up so that the parts behind them start on 16 bytes
static long long table_floats(const MdbTextAttnArgs& a) {
  return a.table != nullptr ? (static_cast<long long>(a.B) * a.H * ((a.Sq + TR - 1) / TR) * a.buckets + 3) / 4 * 4 : 0;
}
long long text_attention_backward_floats(const MdbTextAttnArgs& a) { return table_floats(a) + part_floats(a, text_parts(a)); }

int text_attention_backward(const MdbTextAttnArgs& a, cudaStream_t st) {
  TextParts parts = text_parts(a);
  parts.ws = a.ws + table_floats(a);
  if (int r = a.Dh == 128 ? text_backward<128>(a, parts, st) : text_backward<64>(a, parts, st)) return r;
  const int part_rows = parts.slices > 0 ? std::min(a.sinks, a.Skv) : parts.count > 1 ? a.Skv : 0;
  const long long adders = static_cast<long long>((part_rows + 31) / 32) * a.Hkv * a.B, params = a.d_sink != nullptr || a.d_table != nullptr ? a.H : 0;
  if (adders + params > 0x7fffffff) return -8;
  if (adders + params > 0)
    text_finish_kernel<<<static_cast<unsigned>(adders + params), 256, 0, st>>>(a, parts, part_rows, static_cast<int>(adders), (a.Sq + TR - 1) / TR);
  return static_cast<int>(cudaGetLastError());
}

}  // namespace mdb

MDB_DEFINE_WAIT_LIMIT_SETTER(mdb_set_wait_limit_text_bwd)
