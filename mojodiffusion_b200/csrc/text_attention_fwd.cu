// Forward pass of the language models' attention over a prompt, on tcgen05 / TMEM.
//
//   o_i = sum_j p_ij v_j,  p_ij = exp2(x_ij - m_i) / l_i,  x_ij = log2(e) (scale q_i . k_j + bias(j - i)),  m_i a running reference of x_ij
//
// A CTA owns up to 256 / Dh * 64 query rows, in tiles of 128, that read the same keys and values: the same rows of several heads of one group where the
// group's size allows (they visit the same key tiles, whatever the window), else consecutive rows of one head. Every tile has its softmax
// warpgroup, one thread per row: it turns the scores S = Q K^T (fp32 in TMEM) into probabilities, bf16, written into TMEM over the scores they came
// from and read from there as the A operand of O += P V, while the tensor core works for the other tiles. K and V arrive by TMA.
// Heads of 128: 2 tiles with 128 keys at a time fill the 512 columns of TMEM. Heads of 64: 4 tiles with 64 keys; exponentials bound them, and
// four softmax warps per scheduler instead of two hide their latencies (8 x 512 x 64 x 64 with position buckets: 2 tiles of 128 keys 117 us).
//
// A CTA works through several such items. Its loads and the first scores of the next item run under the epilogue of this one, which needs only O:
// with a window an item has few key tiles, and the start and end of a CTA would be a third of its time.
//
// Key tiles are visited only where a row of the CTA may see a key: the tiles of the first `sinks` keys, then those of the windows. Pieces of 32 keys
// that none of a warp's 32 rows sees are not exponentiated, those that all of them see are not masked; in the others each thread makes
// its row's 32 visibility bits from three bounds.
// BIAS: where all distances of such a piece lie in one bucket, that bias is folded into the exponent's fused multiply-add; in the others the bias of
// element (i, j) is element j - i of a table in shared memory (TextLut).
//
// Rows of V that no row of the CTA sees are zeroed in shared memory before the product, for 0 * NaN is not 0.
#include "text_attention.cuh"
#include "gemm_api.h"

#include <string.h>

namespace mdb {

constexpr int TQ = 128;                              // rows of a query tile

template <int DH> struct FwdShape {
  static constexpr int NT = DH == 64 ? 4 : 2;        // query tiles
  static constexpr int TK = DH == 64 ? 64 : 128;     // keys of a key tile
  static constexpr int STAGES = DH == 64 ? 4 : 2;    // of K and of V
  static constexpr int THREADS = 128 + NT * 128;     // warps 0: TMA, 1 (and 2 with four tiles): MMA issue for two tiles each; four per query tile
  static constexpr int CTRL_REGS = DH == 64 ? 56 : 88, SOFT_REGS = DH == 64 ? 104 : 208;      // 128 ctrl + 128 NT soft <= THREADS * (96, 168)
  static constexpr int Q_BYTES = TQ * DH * 2, K_BYTES = TK * DH * 2;
  static constexpr int Q_BOX = TQ * 128, K_BOX = TK * 128;      // 64 columns of a tile
  static constexpr int BYTES = NT * Q_BYTES + STAGES * 2 * K_BYTES + NT * 4 * 2048 + 1024;
};

struct alignas(64) TextMaps {
  CUtensorMap q, k, v;
};

template <int REGS> __device__ __forceinline__ void regs_up() { asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(REGS)); }
template <int REGS> __device__ __forceinline__ void regs_down() { asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(REGS)); }

// How the query tiles of an item lie: `heads` heads (a divisor of the group's) x `blocks` blocks of rows, both powers of two
struct TextTiles {
  int heads, heads_log, blocks;          // per item
  int row_items, items;       // items along the rows; in all
};

// One work item, seen by a whole warp: its query tiles, and the key tiles that any of them visits: [0, ns) and then [lo, lo + n_kv - ns).
// Lane l looks at query tile l % NT.
template <int DH, bool BIAS> struct TextItem {
  using Shape = FwdShape<DH>;
  static constexpr int NT = Shape::NT, TK = Shape::TK;
  int batch, head, q0;        // of the first tile
  TextSight sight;
  TextKeys all;               // keys that any row sees
  int t_lo, t_hi;             // key tiles of this lane's query tile: [t_lo, t_hi), and of [0, ns) those below t_hi
  int ns, lo, n_kv;

  static __device__ __forceinline__ int tile_head(int head, int t, const TextTiles& l) { return head + (t & (l.heads - 1)); }
  static __device__ __forceinline__ int tile_q0(int q0, int t, const TextTiles& l) { return q0 + (t >> l.heads_log) * TQ; }
  __device__ __forceinline__ void set(const MdbTextAttnArgs& a, int item, const TextTiles& l) {
    int block;
    if (BIAS) {                 // the items of a head follow one another, so that its bias table is made once
      const int rest = item / l.row_items;
      block = item - rest * l.row_items;
      head = rest / a.B;
      batch = rest - head * a.B;
    } else {                    // the last rows, which have the most keys without a window, of all heads and sequences first
      const int groups = a.H >> l.heads_log, rest = item / groups;
      head = (item - rest * groups) << l.heads_log;
      block = rest / a.B;
      batch = rest - block * a.B;
      block = l.row_items - 1 - block;
    }
    q0 = block * l.blocks * TQ;
    sight = text_sight(a, batch);
    const int t = threadIdx.x & (NT - 1), first = tile_q0(q0, t, l);
    TextKeys k = {0, 0, 0};
    if (t < l.heads * l.blocks && first < a.Sq) k = text_keys<BIAS>(a, sight, sight.start + first, sight.start + min(first + TQ, a.Sq) - 1);
    const int n_sinks = (k.sinks + TK - 1) / TK;
    t_lo = k.lo / TK;
    t_hi = max(k.end > k.lo ? (k.end + TK - 1) / TK : 0, n_sinks);
    ns = __reduce_max_sync(0xffffffffu, n_sinks);
    all.end = __reduce_max_sync(0xffffffffu, k.end);
    all.lo = __reduce_min_sync(0xffffffffu, k.end > 0 ? k.lo : 0x7fffffff);
    all.sinks = __reduce_min_sync(0xffffffffu, k.end > 0 ? k.sinks : 0x7fffffff);
    lo = max(all.lo / TK, ns);
    n_kv = all.end == 0 ? 0 : ns + max(__reduce_max_sync(0xffffffffu, t_hi) - lo, 0);
  }
  __device__ __forceinline__ int key_tile(int i) const { return i < ns ? i : i - ns + lo; }
  __device__ __forceinline__ bool sees(int t_lo_, int t_hi_, int i) const {
    const int kt = key_tile(i);
    return i < n_kv && kt < t_hi_ && (kt >= t_lo_ || kt < ns);
  }
};

template <int N> struct Int {
  static constexpr int value = N;
};

template <int DH, bool BIAS>
__global__ void __launch_bounds__(FwdShape<DH>::THREADS, 1)
text_fwd_kernel(const __grid_constant__ TextMaps maps, const __grid_constant__ MdbTextAttnArgs a, const TextTiles tiles) {
  using Shape = FwdShape<DH>;
  constexpr int NT = Shape::NT, TK = Shape::TK, STAGES = Shape::STAGES, PIECES = TK / 32, PARTS = TK / 64;      // parts: P is published 64 keys at a time
  constexpr int DBOX = DH / 64;
  constexpr uint32_t S_COL = 0, O_COL = NT * TK;        // both 256 columns: tile t's scores from t * TK on, its output from 256 + t * DH on
  static_assert(NT * TK == 256 && NT * DH == 256, "TMEM columns");

  extern __shared__ uint8_t smem_raw[];
  __shared__ uint64_t q_full, q_empty, k_full[STAGES], k_empty[STAGES], v_full[STAGES], v_empty[STAGES];
  __shared__ uint64_t s_full[NT], p_full[NT][PARTS], o_full[NT], o_empty[NT];
  __shared__ uint32_t tmem_base_s;
  __shared__ int abort_s;

  const uint32_t raw_addr = smem_u32(smem_raw);
  uint8_t* smem = smem_raw + (((raw_addr + 1023u) & ~1023u) - raw_addr);
  uint8_t* sQ = smem;
  uint8_t* sK = sQ + NT * Shape::Q_BYTES;
  uint8_t* sV = sK + STAGES * Shape::K_BYTES;
  uint8_t* sO = sV + STAGES * Shape::K_BYTES;        // 2 KB per softmax warp: 32 columns of its 32 output rows
  const TextLut lut(sO + NT * 4 * 2048, BIAS ? text_near(a) : 0);

  const int warp = threadIdx.x >> 5;
  const int lane = threadIdx.x & 31;
  // BIAS: a range of items, else every gridDim.x-th
  const int first = BIAS ? static_cast<int>(static_cast<long long>(tiles.items) * blockIdx.x / gridDim.x) : blockIdx.x;
  const int last = BIAS ? static_cast<int>(static_cast<long long>(tiles.items) * (blockIdx.x + 1) / gridDim.x) : tiles.items;
  const int step = BIAS ? 1 : gridDim.x;
  TextItem<DH, BIAS> w;

  if (threadIdx.x == 0) {
    mbar_init(&q_full, 1);
    mbar_init(&q_empty, NT / 2);
    for (int s = 0; s < STAGES; ++s) {
      mbar_init(&k_full[s], 1);
      mbar_init(&k_empty[s], NT / 2);
      mbar_init(&v_full[s], 1);
      mbar_init(&v_empty[s], NT / 2);
    }
    for (int t = 0; t < NT; ++t) {
      mbar_init(&s_full[t], 1);
      for (int h = 0; h < PARTS; ++h) mbar_init(&p_full[t][h], 4);
      mbar_init(&o_full[t], 1);
      mbar_init(&o_empty[t], 4);
    }
    abort_s = 0;
    fence_mbar_init();
  }
  if (warp == 1) {
    tmem_alloc(&tmem_base_s, 512);
    tmem_relinquish();
  }
  if (warp == 0 && lane == 0) {
    tma_prefetch_desc(&maps.q);
    tma_prefetch_desc(&maps.k);
    tma_prefetch_desc(&maps.v);
  }
  if (BIAS) lut.set_buckets(a, threadIdx.x, Shape::THREADS);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem_base = tmem_base_s;

  if (warp < 4) {
    regs_down<Shape::CTRL_REGS>();
    if (warp == 0) {
      // ----------------------------- TMA producer -----------------------------
      const int rep = a.H / a.Hkv, n_q = tiles.heads * tiles.blocks;
      bool ok = true;
      uint64_t* last_bar = nullptr;
      uint32_t last_par = 0;
      int n_items = 0, n_tiles = 0;           // that have keys; key tiles so far
      for (int item = first; ok && item < last; item += step) {
        w.set(a, item, tiles);
        if (w.n_kv == 0) continue;
        ok = __all_sync(0xffffffffu, mbar_wait(&q_empty, (n_items & 1) ^ 1u, &abort_s));
        if (!ok) {
          if (lane == 0) report_status(a.status, STATUS_TIMEOUT, 110, item);
          break;
        }
        if (elect_one()) {
          mbar_expect_tx(&q_full, n_q * Shape::Q_BYTES);
          for (int t = 0; t < n_q; ++t)
            for (int d = 0; d < DBOX; ++d)
              tma_load_4d(sQ + t * Shape::Q_BYTES + d * Shape::Q_BOX, &maps.q, &q_full, d * 64, w.tile_q0(w.q0, t, tiles), w.tile_head(w.head, t, tiles), w.batch);
        }
        __syncwarp();
        last_bar = &q_full;
        last_par = n_items & 1;
        ++n_items;
        const int kv_head = w.head / rep;
        for (int i = 0; ok && i < w.n_kv; ++i, ++n_tiles) {
          const int st = n_tiles % STAGES;
          const uint32_t par = (n_tiles / STAGES) & 1;
          for (int kv = 0; kv < 2; ++kv) {
            uint64_t* empty = kv ? &v_empty[st] : &k_empty[st];
            uint64_t* full = kv ? &v_full[st] : &k_full[st];
            ok = __all_sync(0xffffffffu, mbar_wait(empty, par ^ 1u, &abort_s));
            if (!ok) {
              if (lane == 0) report_status(a.status, STATUS_TIMEOUT, 111 + kv, i);
              break;
            }
            if (elect_one()) {
              mbar_expect_tx(full, Shape::K_BYTES);
              for (int d = 0; d < DBOX; ++d)
                tma_load_4d((kv ? sV : sK) + st * Shape::K_BYTES + d * Shape::K_BOX, kv ? &maps.v : &maps.k, full, d * 64, w.key_tile(i) * TK, kv_head, w.batch);
            }
            __syncwarp();
            last_bar = full;
            last_par = par;
          }
        }
      }
      if (!ok && last_bar != nullptr) {
        const uint64_t t0 = globaltimer_ns();
        while (!mbar_try_wait(last_bar, last_par) && globaltimer_ns() - t0 < 5000000ull) {
        }
      }
    } else if (warp <= NT / 2) {
      // ----------------------------- MMA issue: query tiles t0 and t0 + 1 -----
      // The order of the tensor core's work is this warp's: P V of a tile, then its next S, in turn with the other tile. What a turn takes
      // beside its MMAs delays both, so everything that does not change within an item is at hand.
      const int t0 = (warp - 1) * 2;
      const uint32_t s_col = tmem_base + S_COL + t0 * TK, o_col = tmem_base + O_COL + t0 * DH;
      const uint64_t q_desc = make_desc_kmajor_sw128(smem_u32(sQ + t0 * Shape::Q_BYTES)), k_desc = make_desc_kmajor_sw128(smem_u32(sK));
      const uint64_t v_desc = make_desc_mnmajor_sw128(smem_u32(sV), Shape::K_BOX);
      constexpr uint32_t idesc_s = make_idesc(1, UMMA_BF16, UMMA_BF16, 0, 0, TQ, TK), idesc_pv = make_idesc(1, UMMA_BF16, UMMA_BF16, 0, 1, TQ, DH);
      const auto issue_s = [&](int u, int st) {
#pragma unroll
        for (int kk = 0; kk < DH / 16; ++kk) {
          const uint32_t q_off = u * Shape::Q_BYTES + (kk / 4) * Shape::Q_BOX + (kk % 4) * 32, k_off = (kk / 4) * Shape::K_BOX + (kk % 4) * 32;
          umma_f16_ss(s_col + u * TK, q_desc + (q_off >> 4), k_desc + ((st * Shape::K_BYTES + k_off) >> 4), idesc_s, kk != 0 ? 1u : 0u);
        }
        umma_commit(&s_full[t0 + u]);
      };
      const auto issue_pv = [&](int u, int st, int part, uint32_t more) {
#pragma unroll
        for (int k2 = 0; k2 < 4; ++k2) {
          const int kk = part * 4 + k2;
          umma_f16_ts(o_col + u * DH, s_col + u * TK + kk * 8, v_desc + ((st * Shape::K_BYTES + kk * 2048) >> 4), idesc_pv, kk == 0 ? more : 1u);
        }
      };
      int n_items = 0, n_tiles = 0;
      uint32_t done[2] = {0, 0}, outs[2] = {0, 0};      // key tiles, and items with keys, that either query tile has behind it
      bool ok = true;
      for (int item = first; ok && item < last; item += step) {
        w.set(a, item, tiles);
        if (w.n_kv == 0) continue;
        int t_lo[2], t_hi[2];
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          t_lo[u] = __shfl_sync(0xffffffffu, w.t_lo, t0 + u);
          t_hi[u] = __shfl_sync(0xffffffffu, w.t_hi, t0 + u);
        }
        ok = __all_sync(0xffffffffu, mbar_wait(&q_full, n_items & 1, &abort_s) && mbar_wait(&k_full[n_tiles % STAGES], (n_tiles / STAGES) & 1, &abort_s));
        if (!ok) {
          if (lane == 0) report_status(a.status, STATUS_TIMEOUT, 121, item);
          break;
        }
        ++n_items;
        tc_fence_after();
        if (elect_one()) {
#pragma unroll
          for (int u = 0; u < 2; ++u)
            if (w.sees(t_lo[u], t_hi[u], 0)) issue_s(u, n_tiles % STAGES);
          umma_commit(&k_empty[n_tiles % STAGES]);
          if (w.n_kv == 1) umma_commit(&q_empty);
        }
        __syncwarp();
        // the epilogue of the item before has read the tiles' O
#pragma unroll
        for (int u = 0; u < 2; ++u)
          if (ok && t_hi[u] > 0) ok = __all_sync(0xffffffffu, mbar_wait(&o_empty[t0 + u], (outs[u]++ & 1) ^ 1u, &abort_s));
        if (!ok) {
          if (lane == 0) report_status(a.status, STATUS_TIMEOUT, 122, item);
          break;
        }
        uint32_t begun[2] = {0, 0};
        for (int i = 0; i < w.n_kv; ++i, ++n_tiles) {
          const int st = n_tiles % STAGES, st_n = (n_tiles + 1) % STAGES;
          const bool more = i + 1 < w.n_kv;
          ok = __all_sync(0xffffffffu, mbar_wait(&v_full[st], (n_tiles / STAGES) & 1, &abort_s) &&
                                           (!more || mbar_wait(&k_full[st_n], ((n_tiles + 1) / STAGES) & 1, &abort_s)));
          if (!ok) {
            if (lane == 0) report_status(a.status, STATUS_TIMEOUT, 123, i);
            break;
          }
          const int k0 = w.key_tile(i) * TK;
          if (k0 + TK > w.all.end || (k0 < w.all.lo && k0 + TK > w.all.sinks)) {
#pragma unroll 1
            for (int r = lane; r < TK; r += 32) {
              const int j = k0 + r;
              if (j < w.all.end && (j >= w.all.lo || j < w.all.sinks)) continue;
#pragma unroll 1
              for (int c = 0; c < 8 * DBOX; ++c)
                *reinterpret_cast<uint4*>(sV + st * Shape::K_BYTES + (c >> 3) * Shape::K_BOX + r * 128 + ((c + r) & 7) * 16) = make_uint4(0, 0, 0, 0);
            }
            fence_proxy_async_smem();
            __syncwarp();
          }
          const auto turn = [&](auto which) {
            constexpr int u = decltype(which)::value;
            const bool next = w.sees(t_lo[u], t_hi[u], i + 1);
            if (w.sees(t_lo[u], t_hi[u], i)) {
#pragma unroll
              for (int part = 0; part < PARTS; ++part) {
                ok = __all_sync(0xffffffffu, mbar_wait(&p_full[t0 + u][part], done[u] & 1, &abort_s));
                if (!ok) {
                  if (lane == 0) report_status(a.status, STATUS_TIMEOUT, 124 + t0 + u, i);
                  return;
                }
                tc_fence_after();
                if (elect_one()) {
                  issue_pv(u, st, part, begun[u]);
                  if (part == PARTS - 1) {
                    umma_commit(&o_full[t0 + u]);
                    if (next) issue_s(u, st_n);
                  }
                }
                __syncwarp();
              }
              ++done[u];
              begun[u] = 1;
            } else if (next) {
              if (elect_one()) issue_s(u, st_n);
              __syncwarp();
            }
          };
          turn(Int<0>());
          if (!ok) break;
          turn(Int<1>());
          if (!ok) break;
          if (elect_one()) {
            umma_commit(&v_empty[st]);
            if (more) umma_commit(&k_empty[st_n]);
            if (i + 2 == w.n_kv) umma_commit(&q_empty);
          }
          __syncwarp();
        }
      }
    }
    __syncwarp();
  } else {
    // ------------------------------- softmax: one thread per query row -----------------------
    regs_up<Shape::SOFT_REGS>();
    const int t = (warp - 4) >> 2;
    const int quad = warp & 3;
    const uint32_t lane_addr = static_cast<uint32_t>(quad * 32) << 16;
    const uint32_t s_tile = tmem_base + lane_addr + S_COL + t * TK;
    const uint32_t o_addr = tmem_base + lane_addr + O_COL + t * DH;
    const float sl2 = a.scale * TXT_LOG2E;
    const int near = lut.near;
    uint8_t* stage = sO + (warp - 4) * 2048;
    bool ok = true;
    int done = 0, lut_head = -1;

    for (int item = first; item < last; item += step) {
      w.set(a, item, tiles);
      const int head = w.tile_head(w.head, t, tiles), row0 = w.tile_q0(w.q0, t, tiles) + quad * 32;      // the warp's first row
      if (BIAS && head != lut_head) {
        asm volatile("bar.sync 1, %0;" ::"n"(NT * 128) : "memory");           // nobody reads the head before
        lut.set_head(a, head, threadIdx.x - 128, NT * 128);
        asm volatile("bar.sync 1, %0;" ::"n"(NT * 128) : "memory");
        lut_head = head;
      }
      if (!ok || t >= tiles.heads * tiles.blocks || row0 - quad * 32 >= a.Sq) continue;
      const int my_lo = __shfl_sync(0xffffffffu, w.t_lo, t), my_hi = __shfl_sync(0xffffffffu, w.t_hi, t);
      const int p0 = w.sight.start + row0;        // position of the warp's first row
      // The reference m and the divisor l; a sink logit is the first member of the sum.
      float m_used = -INFINITY, l_run = 0.f;
      if (!BIAS && a.sink_logits != nullptr) {
        m_used = TXT_LOG2E * text_param(a.sink_logits, a.param_f32, head);
        l_run = m_used == -INFINITY ? 0.f : 1.f;
      }
      bool fresh = true;

      for (int i = 0; ok && i < w.n_kv; ++i) {
        if (!w.sees(my_lo, my_hi, i)) continue;
        const int k0 = w.key_tile(i) * TK;
        ok = __all_sync(0xffffffffu, mbar_wait(&s_full[t], done & 1, &abort_s));
        if (!ok) {
          if (lane == 0) report_status(a.status, STATUS_TIMEOUT, 131 + t, i);
          break;
        }
        tc_fence_after();
        uint32_t sv[PIECES][32];
#pragma unroll
        for (int c = 0; c < PIECES; ++c) tmem_ld_32x32b_x32(s_tile + c * 32, sv[c]);
        tmem_wait_ld();
        float mul = sl2, add = 0.f;           // exponent = mul * score + add - m
        if (BIAS) {
          const int d = k0 - row0;
          if (d - 31 >= near) add = lut.behind();
          else if (d + TK - 1 <= -near) add = lut.before();
          else {
            const float* b = lut.from(d - lane);
            mul = 1.f;
#pragma unroll
            for (int c = 0; c < PIECES; ++c)
#pragma unroll
              for (int e = 0; e < 32; e += 4) {
                const float4 u = *reinterpret_cast<const float4*>(b + c * 32 + e);
                const float2 x01 = ffma2(make_float2(__uint_as_float(sv[c][e]), __uint_as_float(sv[c][e + 1])), make_float2(sl2, sl2), make_float2(u.x, u.y));
                const float2 x23 = ffma2(make_float2(__uint_as_float(sv[c][e + 2]), __uint_as_float(sv[c][e + 3])), make_float2(sl2, sl2), make_float2(u.z, u.w));
                sv[c][e] = __float_as_uint(x01.x);
                sv[c][e + 1] = __float_as_uint(x01.y);
                sv[c][e + 2] = __float_as_uint(x23.x);
                sv[c][e + 3] = __float_as_uint(x23.y);
              }
          }
        }
        if (BIAS ? k0 + TK > w.sight.valid : !(k0 + TK - 1 <= p0 && k0 + TK <= w.sight.valid && (k0 > p0 + 31 - a.window || k0 + TK <= a.sinks))) {
#pragma unroll
          for (int c = 0; c < PIECES; ++c) {
            const uint32_t see = BIAS ? bits_below(w.sight.valid - k0 - c * 32) : text_mask(a, w.sight.valid, p0 + lane, k0 + c * 32);
#pragma unroll
            for (int e = 0; e < 32; ++e)
              if (!(see >> e & 1u)) sv[c][e] = 0xff800000u;        // -inf
          }
        }
        float mc[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
        for (int e = 0; e < 32; e += 8 / PIECES)
#pragma unroll
          for (int n = 0; n < 4; ++n) {
            constexpr int PER = 4 / PIECES;                 // chains in a piece
            const int c = n / PER, at = e + 2 * (n % PER);
            mc[n] = fmax3(mc[n], __uint_as_float(sv[c][at]), __uint_as_float(sv[c][at + 1]));
          }
        const float mx = fmaf(fmaxf(fmaxf(mc[0], mc[1]), fmaxf(mc[2], mc[3])), mul, add);
        if (fresh) {
          if (mx > m_used) {
            l_run *= exp2f(m_used - mx);
            m_used = mx;
          }
        } else {
          // The reference is raised when a row has outgrown it by more than 2^8, and with the first key that a row sees.
          const bool need = mx > m_used + 8.0f;
          if (__any_sync(0xffffffffu, need)) {
            ok = __all_sync(0xffffffffu, mbar_wait(&o_full[t], (done - 1) & 1, &abort_s));
            if (!ok) {
              if (lane == 0) report_status(a.status, STATUS_TIMEOUT, 141 + t, i);
              break;
            }
            tc_fence_after();
            const float alpha = need ? exp2f(m_used - mx) : 1.0f;
            if (need) m_used = mx;
            l_run *= alpha;
#pragma unroll 1
            for (int c = 0; c < DH / 16; ++c) {
              uint32_t r[16];
              tmem_ld_32x32b_x16(o_addr + c * 16, r);
              tmem_wait_ld();
#pragma unroll
              for (int e = 0; e < 16; ++e) r[e] = __float_as_uint(__uint_as_float(r[e]) * alpha);
              tmem_st_32x32b_x16(o_addr + c * 16, r);
            }
            tmem_wait_st();
          }
        }
        const float m_now = m_used == -INFINITY ? 0.f : m_used;          // no key so far: every exponent is -inf
        float2 sum_a = make_float2(0.f, 0.f), sum_b = make_float2(0.f, 0.f);
        const float2 mul2 = make_float2(mul, mul), nm2 = make_float2(add - m_now, add - m_now);
#pragma unroll
        for (int c = 0; c < PIECES; ++c) {
          uint32_t pk[16];
#pragma unroll
          for (int e = 0; e < 32; e += 4) {
            // half of every second group of four exponentials runs on the FMA pipe: the special-function unit bounds the rest
            const float2 x01 = ffma2(make_float2(__uint_as_float(sv[c][e]), __uint_as_float(sv[c][e + 1])), mul2, nm2);
            const float2 x23 = ffma2(make_float2(__uint_as_float(sv[c][e + 2]), __uint_as_float(sv[c][e + 3])), mul2, nm2);
            const float2 u = make_float2(ex2_approx(x01.x), ex2_approx(x23.x));
            float2 v;
            if ((e >> 2) % 2 == 1) v = ex2_poly2(make_float2(x01.y, x23.y), -127.f);
            else v = make_float2(ex2_approx(x01.y), ex2_approx(x23.y));
            sum_a = fadd2(sum_a, u);
            sum_b = fadd2(sum_b, v);
            pk[e >> 1] = pack_bf16x2(u.x, v.x);
            pk[(e >> 1) + 1] = pack_bf16x2(u.y, v.y);
          }
          tmem_st_32x32b_x16(s_tile + c * 16, pk);          // over scores that are in registers by now
          if (c & 1) {
            tmem_wait_st();
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(&p_full[t][c >> 1]);
          }
        }
        l_run += (sum_a.x + sum_a.y) + (sum_b.x + sum_b.y);
        ++done;
        fresh = false;
      }
      if (ok && !fresh) {
        ok = __all_sync(0xffffffffu, mbar_wait(&o_full[t], (done - 1) & 1, &abort_s));
        if (!ok && lane == 0) report_status(a.status, STATUS_TIMEOUT, 135 + t, w.n_kv);
      }
      if (!ok) continue;
      tc_fence_after();
      const uint32_t keep = m_used == -INFINITY ? 0u : 0xffffffffu;      // a row without keys is zero whatever O holds
      const float inv_l = 1.f / l_run;
      // 32 columns at a time through shared memory, so that a store covers 64 bytes of eight rows instead of 16 of 32
      __nv_bfloat16* o = static_cast<__nv_bfloat16*>(a.o) + w.batch * a.o_strides[0] + head * a.o_strides[2] + (row0 + (lane >> 2)) * a.o_strides[1] + (lane & 3) * 8;
      const int left = a.Sq - row0 - (lane >> 2);                        // rows of this lane from its first one on
      uint4* mine = reinterpret_cast<uint4*>(stage + lane * 64);
      const uint4* theirs = reinterpret_cast<const uint4*>(stage + (lane >> 2) * 64) + ((lane & 3) ^ (lane >> 3 & 3));
#pragma unroll 1
      for (int c = 0; c < DH / 32; ++c, o += 32) {
        uint32_t r[32];
        if (fresh) {
#pragma unroll
          for (int n = 0; n < 4; ++n)
            if (n * 8 < left) *reinterpret_cast<uint4*>(o + n * 8 * a.o_strides[1]) = make_uint4(0, 0, 0, 0);
          continue;
        }
        tmem_ld_32x32b_x32(o_addr + c * 32, r);
        tmem_wait_ld();
        if (c == DH / 32 - 1) tc_fence_before();
        __syncwarp();
        if (c == DH / 32 - 1 && lane == 0) mbar_arrive(&o_empty[t]);      // the next item's products may have O
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          uint4 v;
          v.x = pack_bf16x2(__uint_as_float(r[8 * e + 0]) * inv_l, __uint_as_float(r[8 * e + 1]) * inv_l) & keep;
          v.y = pack_bf16x2(__uint_as_float(r[8 * e + 2]) * inv_l, __uint_as_float(r[8 * e + 3]) * inv_l) & keep;
          v.z = pack_bf16x2(__uint_as_float(r[8 * e + 4]) * inv_l, __uint_as_float(r[8 * e + 5]) * inv_l) & keep;
          v.w = pack_bf16x2(__uint_as_float(r[8 * e + 6]) * inv_l, __uint_as_float(r[8 * e + 7]) * inv_l) & keep;
          mine[e ^ (lane >> 1 & 3)] = v;
        }
        __syncwarp();
#pragma unroll
        for (int n = 0; n < 4; ++n)
          if (n * 8 < left) *reinterpret_cast<uint4*>(o + n * 8 * a.o_strides[1]) = theirs[n * 32];
      }
      __syncwarp();
      // +inf where a row saw nothing: the backward pass then finds probabilities of zero
      if (a.lse != nullptr && row0 + lane < a.Sq)
        a.lse[(static_cast<long long>(w.batch) * a.H + head) * a.Sq + row0 + lane] = l_run > 0.f && m_used != -INFINITY ? m_used + log2f(l_run) : INFINITY;
    }
  }

  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem_base, 512);
  }
}

static int text_map(CUtensorMap* m, const void* ptr, int B, int S, int H, int Dh, const long long* strides, int rows) {
  int64_t ext[4] = {Dh, S, H, B};
  int64_t str[4] = {2, strides[1] * 2, strides[2] * 2, strides[0] * 2};
  int box[4] = {64, rows, 1, 1};
  return mdb_make_tmap(m, ptr, 2, 4, ext, str, box, 1);
}

template <int DH, bool BIAS>
static int launch_text_fwd(const MdbTextAttnArgs& a, cudaStream_t st) {
  using Shape = FwdShape<DH>;
  TextMaps maps;
  int r = text_map(&maps.q, a.q, a.B, a.Sq, a.H, DH, a.q_strides, TQ);
  if (r) return 1000 + r;
  r = text_map(&maps.k, a.k, a.B, a.Skv, a.Hkv, DH, a.k_strides, Shape::TK);
  if (r) return 2000 + r;
  r = text_map(&maps.v, a.v, a.B, a.Skv, a.Hkv, DH, a.v_strides, Shape::TK);
  if (r) return 3000 + r;
  constexpr int MOST = 226 * 1024;
  auto kern = text_fwd_kernel<DH, BIAS>;
  static bool ready[TXT_DEVICES];
  if ((r = allow_smem(kern, MOST, ready))) return r;
  const int smem = Shape::BYTES + (BIAS ? TextLut::bytes(text_near(a)) : 0);
  if (smem > MOST) return -6;
  // As many tiles to an item as leave an item for every SM, heads of a group before blocks of rows. The bias table in shared memory is one head's.
  const int row_blocks = (a.Sq + TQ - 1) / TQ, sms = device_sm_count();
  TextTiles l;
  long long items = 0;
  for (int n = Shape::NT; n >= 1; n /= 2) {
    l.heads = 1;
    l.heads_log = 0;
    while (!BIAS && 2 * l.heads <= n && (a.H / a.Hkv) % (2 * l.heads) == 0) {
      l.heads *= 2;
      ++l.heads_log;
    }
    l.blocks = n / l.heads;
    l.row_items = (row_blocks + l.blocks - 1) / l.blocks;
    items = static_cast<long long>(l.row_items) * (a.H / l.heads) * a.B;
    if (items >= sms) break;
  }
  if (items > 0x7fffffff) return -8;
  l.items = static_cast<int>(items);
  kern<<<static_cast<unsigned>(items < sms ? items : sms), Shape::THREADS, smem, st>>>(maps, a, l);
  return static_cast<int>(cudaGetLastError());
}

int text_attention_prompt(const MdbTextAttnArgs& a, cudaStream_t st) {
  if (a.table != nullptr) return a.Dh == 128 ? launch_text_fwd<128, true>(a, st) : launch_text_fwd<64, true>(a, st);
  return a.Dh == 128 ? launch_text_fwd<128, false>(a, st) : launch_text_fwd<64, false>(a, st);
}

}  // namespace mdb

MDB_DEFINE_WAIT_LIMIT_SETTER(mdb_set_wait_limit_text_fwd)
