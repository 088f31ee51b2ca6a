// Forward pass of the language models' attention over a prompt, on tcgen05 / TMEM.
//
//   o_i = sum_j p_ij v_j,  p_ij = exp2(x_ij - m_i) / l_i,  x_ij = log2(e) (scale q_i . k_j + bias(j - i)),  m_i a running reference of x_ij
//
// A CTA owns two tiles of 128 query rows that read the same keys and values: the same rows of two heads of one group where the group's size is even
// (they visit the same key tiles, whatever the window), else 256 consecutive rows of one head. Either tile has its softmax warpgroup, one thread
// per row: it turns the scores S = Q K^T (fp32 in TMEM) into probabilities, bf16, written into TMEM over the scores they came from and read from
// there as the A operand of O += P V, while the tensor core works for the other tile. K and V arrive by TMA.
//
// Heads of 128: 128 keys at a time, which fills TMEM and most of the shared memory with one CTA. It works through several such items: the loads and
// the first scores of the next one run under the epilogue, which needs only O (with a window an item has few key tiles).
// Heads of 64: 64 keys at a time and half of TMEM, so that two CTAs share an SM. There the exponentials and their latencies bound: four softmax warps
// per scheduler instead of two, and the start and the epilogue of one CTA run under the other's work.
//
// Key tiles are visited only where a row of the CTA may see a key: the tiles of the first `sinks` keys, then those of the windows. In a tile that a
// warp's 32 rows do not see whole, each thread makes its row's 32 visibility bits of a piece of 32 keys from three bounds; a piece that all of them see
// is left as it is. Masked pieces go through the exponentials like the others.
// BIAS: where all distances of a warp's rows and a tile lie in one bucket, that bias is folded into the exponent's fused multiply-add; in the other
// tiles the bias of element (i, j) is element j - i of a table in shared memory (TextLut).
//
// Rows of V that no row of the CTA sees are zeroed in shared memory before the product, for 0 * NaN is not 0.
//
// Probabilities go into their product as one bf16 term: they are off by 2^-9 of themselves at most, each in its own direction, as much as the output's own rounding (relative errors against 64
// bits 0.0020 with one term, 0.0016 with two or with fp32). A second term is a second product of the same size: six prompts (below) would take 361 us instead of 268, captions 39.3 instead of 36.5.
// FINE (packed, with a backward pass to come): in sequences whose rows have few keys (see text_is_fine) a probability goes into its product as two bf16 terms, the second one in the half of
// the scores' columns that the first leaves free.
//
// PACKED: an item is a unit of one sequence (see text_unit); coordinates and rows count from the sequence's first row. A tile holds rows of one sequence only, at the cost of tiles that are
// not full: rows of several sequences in a tile would multiply each other's values by zero, and 0 * NaN would carry one sequence's NaN into another. 10155 tokens in six sequences of 301
// to 4096, 32 / 8 heads of 128: 294 us among other passes, 268 by itself (784 and 860 TFLOP/s; equal lengths take 1.01 to 1.05 of the batched form's time; 396 bytes spilled, 340 without sequences); 16 sequences of 7 to 300, 64 / 8 heads of 64, window 128: 33 us,
// a CTA with one key tile 6.7 us of which 2.6 before its first scores.
//
// What bounds it: the latency of a tile's way from the scores through the softmax to the next product; no unit is busy half of the time. 8192 tokens,
// 32 / 8 heads of 128, window 1024 with 4 first keys: 162 us, 797 TFLOP/s of visible pairs, 985 with the masked 19 % of the tiles (tensor pipe active 46 % of
// the cycles, issue slots 43 %, special-function unit 35 %). 8 x 512 tokens, 64 heads of 64 with a table: 80 us, 320 TFLOP/s (17 %, 43 %, 36 %); one CTA
// per SM and 128-key tiles took 100 there, and 199 in the former with a CTA per item instead of a loop over them.
#include "text_attention.cuh"
#include "gemm_api.h"

#include <string.h>

namespace mdb {

constexpr int TQ = 128;                              // rows of a query tile

template <int DH> struct FwdShape {
  static constexpr int TK = DH == 64 ? 64 : 128;     // keys of a key tile
  static constexpr int STAGES = DH == 64 ? 3 : 2;    // of K and of V
  static constexpr int CTAS = DH == 64 ? 2 : 1;      // per SM
  // warps 0: TMA, 1: MMA issue; from SOFT on four per query tile. One CTA per SM has registers to move from a first warpgroup (of which two warps idle).
  static constexpr int SOFT = DH == 64 ? 2 : 4, THREADS = (SOFT + 8) * 32;
  static constexpr int CTRL_REGS = 88, SOFT_REGS = 208;      // 128 ctrl + 256 soft <= 384 * 168
  static constexpr int TMEM = 2 * TK + 2 * DH;       // tile t's scores from t * TK on, its output from 2 * TK + t * DH on
  static constexpr int Q_BYTES = TQ * DH * 2, K_BYTES = TK * DH * 2;
  static constexpr int Q_BOX = TQ * 128, K_BOX = TK * 128;      // 64 columns of a tile
  static constexpr int BYTES = 2 * Q_BYTES + STAGES * 2 * K_BYTES + 8 * 2048 + 1024;
};

struct alignas(64) TextMaps {
  CUtensorMap q, k, v;
};

template <int REGS> __device__ __forceinline__ void regs_up() { asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(REGS)); }
template <int REGS> __device__ __forceinline__ void regs_down() { asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(REGS)); }

// How the query tiles of an item lie: `heads` heads (a divisor of the group's) x `blocks` blocks of rows, both powers of two
struct TextTiles {
  int heads, heads_log, blocks;          // per item: two heads, two blocks, or one of each
  int row_items, items;       // items along the rows; in all
};

// One work item, seen by a whole warp: its query tiles, and the key tiles that any of them visits: [0, ns) and then [lo, lo + n_kv - ns).
// Lane l looks at query tile l % 2.
template <int DH, bool BIAS, bool PACKED, bool FINE> struct TextItem {
  using Shape = FwdShape<DH>;
  static constexpr int TK = Shape::TK;
  int batch, head, q0;        // of the first tile
  int base, rows;             // packed: first row and length of the sequence; else 0 and Sq
  TextSight sight;
  TextKeys all;               // keys that any row sees
  int t_lo, t_hi;             // key tiles of this lane's query tile: [t_lo, t_hi), and of [0, ns) those below t_hi
  int ns, lo, n_kv;

  static __device__ __forceinline__ int tile_head(int head, int t, const TextTiles& l) { return head + (t & (l.heads - 1)); }
  static __device__ __forceinline__ int tile_q0(int q0, int t, const TextTiles& l) { return q0 + (t >> l.heads_log) * TQ; }
  // the order of the items with BIAS: those of a head follow one another, so that its bias table is made once
  static __device__ __forceinline__ int head_of(const MdbTextAttnArgs& a, int item, const TextTiles& l) { return item / l.row_items / a.B; }
  __device__ __forceinline__ void set(const MdbTextAttnArgs& a, int item, const TextTiles& l) {
    TextUnit u = {0, a.Sq, 0};
    if (PACKED) u = text_unit(a, item / (a.H >> l.heads_log), l.blocks * TQ);
    set(a, item, l, u);
  }
  // `u`: packed, the item's unit
  __device__ __forceinline__ void set(const MdbTextAttnArgs& a, int item, const TextTiles& l, const TextUnit& u) {
    int block;
    base = 0;
    rows = a.Sq;
    if (PACKED) {
      const int groups = a.H >> l.heads_log, rest = item / groups;
      head = (item - rest * groups) << l.heads_log;
      batch = 0;
      base = u.base;
      rows = u.rows;
      block = u.block;
    } else if (BIAS) {
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
    if (PACKED) sight = {rows, 0};
    else sight = text_sight(a, batch);
    const int t = threadIdx.x & 1, first = tile_q0(q0, t, l);
    TextKeys k = {0, 0, 0};
    if (t < l.heads * l.blocks && first < rows) k = text_keys<BIAS>(a, sight, sight.start + first, sight.start + min(first + TQ, rows) - 1);
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

template <int DH, bool BIAS, bool PACKED, bool FINE>
__global__ void __launch_bounds__(FwdShape<DH>::THREADS, FwdShape<DH>::CTAS)
text_fwd_kernel(const __grid_constant__ TextMaps maps, const __grid_constant__ MdbTextAttnArgs a, const TextTiles tiles) {
  using Shape = FwdShape<DH>;
  constexpr int TK = Shape::TK, STAGES = Shape::STAGES, PIECES = TK / 32, PARTS = TK / 64;      // parts: P is published 64 keys at a time
  constexpr int DBOX = DH / 64;
  constexpr uint32_t O_COL = 2 * TK;

  extern __shared__ uint8_t smem_raw[];
  __shared__ uint64_t q_full, q_empty, k_full[STAGES], k_empty[STAGES], v_full[STAGES], v_empty[STAGES];
  __shared__ uint64_t s_full[2], p_full[2][PARTS], o_full[2], o_empty[2];
  __shared__ uint32_t tmem_base_s;
  __shared__ int abort_s;

  const uint32_t raw_addr = smem_u32(smem_raw);
  uint8_t* smem = smem_raw + (((raw_addr + 1023u) & ~1023u) - raw_addr);
  uint8_t* sQ = smem;
  uint8_t* sK = sQ + 2 * Shape::Q_BYTES;
  uint8_t* sV = sK + STAGES * Shape::K_BYTES;
  uint8_t* sO = sV + STAGES * Shape::K_BYTES;        // 2 KB per softmax warp: 32 columns of its 32 output rows
  const TextLut lut(sO + 8 * 2048, BIAS ? text_near(a) : 0);

  const int warp = threadIdx.x >> 5;
  const int lane = threadIdx.x & 31;
  // one item to a CTA where two share an SM (the next one starts wherever a CTA ends); else a range of them with BIAS, or every gridDim.x-th
  constexpr bool ONE = Shape::CTAS == 2, RANGE = BIAS && !ONE;
  const int first = RANGE ? static_cast<int>(static_cast<long long>(tiles.items) * blockIdx.x / gridDim.x) : blockIdx.x;
  const int last = ONE ? first + 1 : RANGE ? static_cast<int>(static_cast<long long>(tiles.items) * (blockIdx.x + 1) / gridDim.x) : tiles.items;
  const int step = ONE || RANGE ? 1 : gridDim.x;
  TextItem<DH, BIAS, PACKED, FINE> w;

  const auto clear_rows = [&](bool look, int thread, int threads) {      // packed, rows of no sequence: zero, and no gradient
    text_rows_of_none(a, look, blockIdx.x, gridDim.x, [&](int row) {
      for (int e = thread; e < a.H * (DH / 8); e += threads) {
        const long long to = row * a.o_strides[1] + e / (DH / 8) * a.o_strides[2] + e % (DH / 8) * 8;
        *reinterpret_cast<uint4*>(static_cast<__nv_bfloat16*>(a.o) + to) = make_uint4(0, 0, 0, 0);
        if (a.o_low != nullptr) *reinterpret_cast<uint4*>(static_cast<__nv_bfloat16*>(a.o_low) + to) = make_uint4(0, 0, 0, 0);
        if (a.lse != nullptr && e < a.H) a.lse[static_cast<long long>(e) * a.Sq + row] = INFINITY;
      }
    });
  };
  TextUnit only = {0, 0, 0};  // PACKED, one item to a CTA: its unit. There may be fewer units than the grid has room for
  if (PACKED && ONE) {
    only = text_unit(a, first / (a.H >> tiles.heads_log), tiles.blocks * TQ);
    if (only.rows == 0) {
      clear_rows(true, threadIdx.x, Shape::THREADS);
      return;
    }
  }
  const auto set_first = [&](int item) {
    if (PACKED && ONE) w.set(a, item, tiles, only);
    else w.set(a, item, tiles);
  };

  // The TMA warp makes the barriers and starts loading while the others get ready: nobody else touches either before __syncthreads.
  if (warp == 0) {
    if (lane == 0) {
      tma_prefetch_desc(&maps.q);
      tma_prefetch_desc(&maps.k);
      tma_prefetch_desc(&maps.v);
      mbar_init(&q_full, 1);
      mbar_init(&q_empty, 1);
      for (int s = 0; s < STAGES; ++s) {
        mbar_init(&k_full[s], 1);
        mbar_init(&k_empty[s], 1);
        mbar_init(&v_full[s], 1);
        mbar_init(&v_empty[s], 1);
      }
      for (int t = 0; t < 2; ++t) {
        mbar_init(&s_full[t], 1);
        for (int h = 0; h < PARTS; ++h) mbar_init(&p_full[t][h], 4);
        mbar_init(&o_full[t], 1);
        mbar_init(&o_empty[t], 4);
      }
      abort_s = 0;
      fence_mbar_init();
    }
    __syncwarp();
  } else if (warp == 1) {
    tmem_alloc(&tmem_base_s, Shape::TMEM);
    tmem_relinquish();
  }
  const auto load_q = [&]() {
    const int n_q = tiles.heads * tiles.blocks;
    if (elect_one()) {
      mbar_expect_tx(&q_full, n_q * Shape::Q_BYTES);
#pragma unroll 1
      for (int t = 0; t < n_q; ++t)
        for (int d = 0; d < DBOX; ++d)
          tma_load_4d(sQ + t * Shape::Q_BYTES + d * Shape::Q_BOX, &maps.q, &q_full, d * 64, w.base + w.tile_q0(w.q0, t, tiles), w.tile_head(w.head, t, tiles), w.batch);
    }
    __syncwarp();
  };
  const auto load_kv = [&](int kv, int st, int i, int kv_head) {
    uint64_t* full = kv ? &v_full[st] : &k_full[st];
    if (elect_one()) {
      mbar_expect_tx(full, Shape::K_BYTES);
      for (int d = 0; d < DBOX; ++d)
        tma_load_4d((kv ? sV : sK) + st * Shape::K_BYTES + d * Shape::K_BOX, kv ? &maps.v : &maps.k, full, d * 64, w.base + w.key_tile(i) * TK, kv_head, w.batch);
    }
    __syncwarp();
  };
  const int rep = a.H / a.Hkv;
  int early = 0;              // key tiles of the first item that are on their way
  if (warp == 0 && first < last) {
    set_first(first);
    if (w.n_kv > 0) {
      load_q();
#pragma unroll 1
      for (; early < STAGES && early < w.n_kv; ++early)
#pragma unroll 1
        for (int kv = 0; kv < 2; ++kv) load_kv(kv, early, early, w.head / rep);
    }
  }
  if (BIAS && ONE && warp != 0) lut.set(a, w.head_of(a, first, tiles), warp - 1, Shape::THREADS / 32 - 1);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem_base = tmem_base_s;

  if (warp < Shape::SOFT) {
    if (Shape::CTAS == 1) regs_down<Shape::CTRL_REGS>();
    if (warp == 0) {
      // ----------------------------- TMA producer -----------------------------
      bool ok = true;
      int n_items = 0, n_tiles = 0, loads = 2 * early;           // items that have keys; key tiles so far; loads of K and V in turn
      for (int item = first; ok && item < last; item += step) {
        if (item != first) w.set(a, item, tiles);
        if (w.n_kv == 0) continue;
        if (item != first) {
          ok = text_wait<DH == 128>(&q_empty, (n_items & 1) ^ 1u, &abort_s);
          if (!ok) break;
          load_q();
        }
        ++n_items;
        const int kv_head = w.head / rep;
        for (int i = 0; ok && i < w.n_kv; ++i, ++n_tiles) {
          if (n_tiles < early) continue;
          const int st = n_tiles % STAGES;
          const uint32_t par = (n_tiles / STAGES) & 1;
#pragma unroll 1
          for (int kv = 0; kv < 2; ++kv) {
            ok = text_wait<DH == 128>(kv ? &v_empty[st] : &k_empty[st], par ^ 1u, &abort_s);
            if (!ok) break;
            load_kv(kv, st, i, kv_head);
            ++loads;
          }
        }
      }
      if (!ok) {
        if (lane == 0) report_status(a.status, STATUS_TIMEOUT, 111, n_tiles);
        // The copies on the way land before the memory is given up: the last Q, and the last K and V of every stage. They end in any order.
        for (int j = max(loads - 2 * STAGES, 0) - 1; j < loads; ++j) {
          const bool q = j < max(loads - 2 * STAGES, 0);
          if (q && n_items == 0) continue;
          uint64_t* bar = q ? &q_full : (j & 1 ? v_full : k_full) + (j >> 1) % STAGES;
          const uint32_t par = (q ? n_items - 1 : (j >> 1) / STAGES) & 1;
          const uint64_t t0 = globaltimer_ns();
          while (!mbar_try_wait(bar, par) && globaltimer_ns() - t0 < 5000000ull) {
          }
        }
      }
    } else if (warp == 1) {
      // ----------------------------- MMA issue --------------------------------
      // The order of the tensor core's work is this warp's: P V of a tile, then its next S, in turn with the other tile. What a turn takes
      // beside its MMAs delays both, so everything that does not change within an item is at hand.
      const uint32_t s_col = tmem_base, o_col = tmem_base + O_COL;
      const uint64_t q_desc = make_desc_kmajor_sw128(smem_u32(sQ)), k_desc = make_desc_kmajor_sw128(smem_u32(sK));
      const uint64_t v_desc = make_desc_mnmajor_sw128(smem_u32(sV), Shape::K_BOX);
      constexpr uint32_t idesc_s = make_idesc(1, UMMA_BF16, UMMA_BF16, 0, 0, TQ, TK), idesc_pv = make_idesc(1, UMMA_BF16, UMMA_BF16, 0, 1, TQ, DH);
      const auto issue_s = [&](int u, int st) {
#pragma unroll
        for (int kk = 0; kk < DH / 16; ++kk) {
          const uint32_t q_off = u * Shape::Q_BYTES + (kk / 4) * Shape::Q_BOX + (kk % 4) * 32, k_off = (kk / 4) * Shape::K_BOX + (kk % 4) * 32;
          umma_f16_ss(s_col + u * TK, q_desc + (q_off >> 4), k_desc + ((st * Shape::K_BYTES + k_off) >> 4), idesc_s, kk != 0 ? 1u : 0u);
        }
        umma_commit(&s_full[u]);
      };
      const auto issue_pv = [&](int u, int st, int part, uint32_t more, bool fine) {
#pragma unroll
        for (int k2 = 0; k2 < 4; ++k2) {
          const int kk = part * 4 + k2;
          umma_f16_ts(o_col + u * DH, s_col + u * TK + kk * 8, v_desc + ((st * Shape::K_BYTES + kk * 2048) >> 4), idesc_pv, kk == 0 ? more : 1u);
        }
        if (FINE && fine) {
          // not unrolled: the addresses of its operands would take registers from every turn of this warp (training case of nine sequences: the kernel 98 us instead of 91)
#pragma unroll 1
          for (int k2 = 0; k2 < 4; ++k2) {
            const int kk = part * 4 + k2;
            umma_f16_ts(o_col + u * DH, s_col + u * TK + TK / 2 + kk * 8, v_desc + ((st * Shape::K_BYTES + kk * 2048) >> 4), idesc_pv, 1u);
          }
        }
      };
      int n_items = 0, n_tiles = 0;
      uint32_t done[2] = {0, 0}, outs[2] = {0, 0};      // key tiles, and items with keys, that either query tile has behind it
      bool ok = true;
      for (int item = first; ok && item < last; item += step) {
        set_first(item);
        if (w.n_kv == 0) continue;
        int t_lo[2], t_hi[2];
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          t_lo[u] = __shfl_sync(0xffffffffu, w.t_lo, u);
          t_hi[u] = __shfl_sync(0xffffffffu, w.t_hi, u);
        }
        ok = text_wait<DH == 128>(&q_full, n_items & 1, &abort_s) && text_wait<DH == 128>(&k_full[n_tiles % STAGES], (n_tiles / STAGES) & 1, &abort_s);
        if (!ok) break;
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
          if (ok && !ONE && t_hi[u] > 0) ok = text_wait<DH == 128>(&o_empty[u], (outs[u]++ & 1) ^ 1u, &abort_s);
        if (!ok) break;
        uint32_t begun[2] = {0, 0};
        const bool fine = FINE && text_is_fine(a, w.rows);
        for (int i = 0; i < w.n_kv; ++i, ++n_tiles) {
          const int st = n_tiles % STAGES, st_n = (n_tiles + 1) % STAGES;
          const bool more = i + 1 < w.n_kv;
          ok = text_wait<DH == 128>(&v_full[st], (n_tiles / STAGES) & 1, &abort_s) && (!more || text_wait<DH == 128>(&k_full[st_n], ((n_tiles + 1) / STAGES) & 1, &abort_s));
          if (!ok) break;
          const int k0 = w.key_tile(i) * TK;
          if (k0 + TK > w.all.end || (k0 < w.all.lo && k0 + TK > w.all.sinks)) {
#pragma unroll 1
            for (int r = lane; r < TK; r += 32) {
              const int j = k0 + r;
              if (j < w.all.end && (j >= w.all.lo || j < w.all.sinks)) continue;
#pragma unroll
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
                ok = text_wait<DH == 128>(&p_full[u][part], done[u] & 1, &abort_s);
                if (!ok) return;
                tc_fence_after();
                if (elect_one()) {
                  issue_pv(u, st, part, begun[u], fine);
                  if (part == PARTS - 1) {
                    umma_commit(&o_full[u]);
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
      if (!ok && lane == 0) report_status(a.status, STATUS_TIMEOUT, 121, n_tiles);
    }
    __syncwarp();
  } else {
    // ------------------------------- softmax: one thread per query row -----------------------
    if (Shape::CTAS == 1) regs_up<Shape::SOFT_REGS>();
    const int t = (warp - Shape::SOFT) >> 2;
    const int quad = warp & 3;
    const uint32_t lane_addr = static_cast<uint32_t>(quad * 32) << 16;
    const uint32_t s_tile = tmem_base + lane_addr + t * TK;
    const uint32_t o_addr = tmem_base + lane_addr + O_COL + t * DH;
    const float sl2 = a.scale * TXT_LOG2E;
    uint8_t* stage = sO + (warp - Shape::SOFT) * 2048;
    bool ok = true;
    int done = 0, lut_head = -1;

    if (first < last) set_first(first);
    for (int item = first; item < last; item += step) {
      const int batch = w.batch, head = w.tile_head(w.head, t, tiles), row0 = w.tile_q0(w.q0, t, tiles) + quad * 32;      // the warp's first row
      const int base = w.base, rows = w.rows;
      if (BIAS && !ONE && head != lut_head) {
        asm volatile("bar.sync 1, 256;" ::: "memory");           // nobody reads the head before
        lut.set(a, head, warp - Shape::SOFT, 8);
        asm volatile("bar.sync 1, 256;" ::: "memory");
        lut_head = head;
      }
      if (!ok || t >= tiles.heads * tiles.blocks || row0 - quad * 32 >= rows) {
        if (item + step < last) w.set(a, item + step, tiles);
        continue;
      }
      const int my_lo = __shfl_sync(0xffffffffu, w.t_lo, t), my_hi = __shfl_sync(0xffffffffu, w.t_hi, t);
      const int p0 = w.sight.start + row0;        // position of the warp's first row
      // key tiles from whole_lo (or below the first keys' end) to whole_hi are seen whole by the warp's rows
      const int valid = w.sight.valid, whole_hi = BIAS ? valid - TK : min(p0 + 1, valid) - TK, whole_lo = BIAS ? 0 : p0 + 32 - a.window;
      // The reference m and the divisor l; a sink logit is the first member of the sum.
      float m_used = -INFINITY, l_run = 0.f;
      if (!BIAS && a.sink_logits != nullptr) {
        m_used = TXT_LOG2E * text_param(a.sink_logits, a.param_f32, head);
        l_run = m_used == -INFINITY ? 0.f : 1.f;
      }
      bool fresh = true;

      if constexpr (FINE) {
        if (text_is_fine(a, rows)) {
          constexpr bool TWO = true;
#include "text_attention_fwd_tiles.cuh"
        } else {
          constexpr bool TWO = false;
#include "text_attention_fwd_tiles.cuh"
        }
      } else {
        constexpr bool TWO = false;
#include "text_attention_fwd_tiles.cuh"
      }
      if (item + step < last) w.set(a, item + step, tiles);      // while the last products run
      if (ok && !fresh) {
        ok = text_wait<DH == 128>(&o_full[t], (done - 1) & 1, &abort_s);
      }
      if (!ok) continue;
      tc_fence_after();
      const uint32_t keep = m_used == -INFINITY ? 0u : 0xffffffffu;      // a row without keys is zero whatever O holds
      const float inv_l = 1.f / l_run;
      // 32 columns at a time through shared memory, so that a store covers 64 bytes of eight rows instead of 16 of 32
      __nv_bfloat16* o = static_cast<__nv_bfloat16*>(a.o) + batch * a.o_strides[0] + head * a.o_strides[2] + (base + row0 + (lane >> 2)) * a.o_strides[1] + (lane & 3) * 8;
      const int left = rows - row0 - (lane >> 2);                        // rows of this lane from its first one on
      uint4* mine = reinterpret_cast<uint4*>(stage + lane * 64);
      const uint4* theirs = reinterpret_cast<const uint4*>(stage + (lane >> 2) * 64) + ((lane & 3) ^ (lane >> 3 & 3));
#pragma unroll 1
      for (int c = 0; c < DH / 32; ++c, o += 32) {
        uint32_t r[32];
        if (fresh) {
#pragma unroll
          for (int n = 0; n < 4; ++n)
            if (n * 8 < left) {
              *reinterpret_cast<uint4*>(o + n * 8 * a.o_strides[1]) = make_uint4(0, 0, 0, 0);
              if (a.o_low != nullptr) *reinterpret_cast<uint4*>(o + (static_cast<__nv_bfloat16*>(a.o_low) - static_cast<__nv_bfloat16*>(a.o)) + n * 8 * a.o_strides[1]) = make_uint4(0, 0, 0, 0);
            }
          continue;
        }
        tmem_ld_32x32b_x32(o_addr + c * 32, r);
        tmem_wait_ld();
        if (c == DH / 32 - 1) tc_fence_before();
        __syncwarp();
        if (!ONE && c == DH / 32 - 1 && lane == 0) mbar_arrive(&o_empty[t]);      // the next item's products may have O
        // the output, and in a second turn what its rounding left
#pragma unroll 1
        for (int low = 0;; ++low) {
          uint32_t v[16];
#pragma unroll
          for (int e = 0; e < 16; ++e) {
            const float x = __uint_as_float(r[2 * e]) * inv_l, y = __uint_as_float(r[2 * e + 1]) * inv_l;
            v[e] = pack_bf16x2(x, y);
            if (low) {
              const float2 h = unpack_bf16x2(v[e]);
              v[e] = pack_bf16x2(x - h.x, y - h.y);
            }
            v[e] &= keep;
          }
#pragma unroll
          for (int e = 0; e < 4; ++e) mine[e ^ (lane >> 1 & 3)] = make_uint4(v[4 * e], v[4 * e + 1], v[4 * e + 2], v[4 * e + 3]);
          __syncwarp();
          __nv_bfloat16* to = low ? o + (static_cast<__nv_bfloat16*>(a.o_low) - static_cast<__nv_bfloat16*>(a.o)) : o;
#pragma unroll
          for (int n = 0; n < 4; ++n)
            if (n * 8 < left) *reinterpret_cast<uint4*>(to + n * 8 * a.o_strides[1]) = theirs[n * 32];
          if (a.o_low == nullptr || low) break;
          __syncwarp();
        }
      }
      __syncwarp();
      // +inf where a row saw nothing: the backward pass then finds probabilities of zero
      if (a.lse != nullptr && row0 + lane < rows)
        a.lse[(static_cast<long long>(batch) * a.H + head) * a.Sq + base + row0 + lane] = m_used == -INFINITY || l_run == 0.f ? INFINITY : m_used + log2f(l_run);
    }
    if (PACKED) clear_rows(!ONE, threadIdx.x - Shape::SOFT * 32, 256);
    if (!ok && lane == 0) report_status(a.status, STATUS_TIMEOUT, 131 + t, done);
  }

  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem_base, Shape::TMEM);
  }
}

static int text_map(CUtensorMap* m, const void* ptr, int B, int S, int H, int Dh, const long long* strides, int rows) {
  int64_t ext[4] = {Dh, S, H, B};
  int64_t str[4] = {2, strides[1] * 2, strides[2] * 2, strides[0] * 2};
  int box[4] = {64, rows, 1, 1};
  return mdb_make_tmap(m, ptr, 2, 4, ext, str, box, 1);
}

template <int DH, bool BIAS, bool PACKED, bool FINE>
static int launch_text_fwd(const MdbTextAttnArgs& a, cudaStream_t st) {
  const int B = PACKED ? 1 : a.B;
  using Shape = FwdShape<DH>;
  TextMaps maps;
  int r = text_map(&maps.q, a.q, B, a.Sq, a.H, DH, a.q_strides, TQ);
  if (r) return 1000 + r;
  r = text_map(&maps.k, a.k, B, a.Skv, a.Hkv, DH, a.k_strides, Shape::TK);
  if (r) return 2000 + r;
  r = text_map(&maps.v, a.v, B, a.Skv, a.Hkv, DH, a.v_strides, Shape::TK);
  if (r) return 3000 + r;
  constexpr int MOST = 226 * 1024;
  auto kern = text_fwd_kernel<DH, BIAS, PACKED, FINE>;
  static bool ready[TXT_DEVICES];
  if ((r = allow_smem(kern, MOST, ready))) return r;
  const int smem = Shape::BYTES + (BIAS ? TextLut::bytes(text_near(a)) : 0);
  if (smem > MOST) return -6;
  // Two tiles to an item unless one leaves fewer SMs idle, heads of a group before blocks of rows. The bias table in shared memory is one head's.
  const int row_blocks = (a.Sq + TQ - 1) / TQ, slots = Shape::CTAS * device_sm_count();
  TextTiles l;
  long long items = 0;
  for (int n = 2; n >= 1; n /= 2) {
    l.heads = 1;
    l.heads_log = 0;
    while (!BIAS && 2 * l.heads <= n && (a.H / a.Hkv) % (2 * l.heads) == 0) {
      l.heads *= 2;
      ++l.heads_log;
    }
    l.blocks = n / l.heads;
    l.row_items = PACKED ? static_cast<int>(text_units(a, l.blocks * TQ)) : (row_blocks + l.blocks - 1) / l.blocks;
    items = static_cast<long long>(l.row_items) * (a.H / l.heads) * B;
    if (items >= slots) break;
  }
  if (items > 0x7fffffff) return -8;
  l.items = static_cast<int>(items);
  if (PACKED && (r = text_make_units(a, l.blocks * TQ, st))) return r;
  kern<<<static_cast<unsigned>(Shape::CTAS == 2 || items < slots ? items : slots), Shape::THREADS, smem, st>>>(maps, a, l);
  return static_cast<int>(cudaGetLastError());
}

int text_attention_prompt(const MdbTextAttnArgs& a, cudaStream_t st) {
  if (a.cu != nullptr) {
    if (a.o_low != nullptr) return a.Dh == 128 ? launch_text_fwd<128, false, true, true>(a, st) : launch_text_fwd<64, false, true, true>(a, st);
    return a.Dh == 128 ? launch_text_fwd<128, false, true, false>(a, st) : launch_text_fwd<64, false, true, false>(a, st);
  }
  if (a.table != nullptr) return a.Dh == 128 ? launch_text_fwd<128, true, false, false>(a, st) : launch_text_fwd<64, true, false, false>(a, st);
  return a.Dh == 128 ? launch_text_fwd<128, false, false, false>(a, st) : launch_text_fwd<64, false, false, false>(a, st);
}

}  // namespace mdb

MDB_DEFINE_WAIT_LIMIT_SETTER(mdb_set_wait_limit_text_fwd)
