// Forward pass of the language models' attention over a prompt, on tcgen05 / TMEM.
//
//   o_i = sum_j p_ij v_j,  p_ij = exp2(x_ij - m_i) / l_i,  x_ij = log2(e) (scale q_i . k_j + bias(j - i)),  m_i a running reference of x_ij
//
// One CTA owns two 128-row query tiles that read the same keys and values: the same rows of two query heads of one key head where a group
// has an even number of heads, else 256 consecutive rows of one head. The tensor core computes one tile's S = Q K^T (128 x 128, fp32 in TMEM)
// and O += P V while the other tile's four softmax warps, one thread per row, turn scores into probabilities: bf16, written into TMEM over
// the scores they came from, read from there as the A operand. K and V tiles arrive by TMA, double buffered.
//
// Key tiles are visited only where a row of the CTA may see a key: the tiles of the first `sinks` keys, then those of the windows. A tile that
// every row sees whole is not masked; in the others each thread makes its row's 128 visibility bits from three bounds.
// BIAS: tiles all of whose distances lie in one bucket (most of a long prompt) fold that bias into the constant of the exponent's fused
// multiply-add; in the others the bias of element (i, j) is element j - i of a table in shared memory, read by 32 lanes at 32 consecutive places.
//
// Rows of V that no row of the CTA sees are zeroed in shared memory before the product, for 0 * NaN is not 0.
#include "text_attention.cuh"
#include "gemm_api.h"

#include <string.h>

namespace mdb {

constexpr int TF_THREADS = 384;                      // warps 0: TMA, 1: MMA issue, 2-3 idle; 4-7 / 8-11: softmax of tile 0 / 1
constexpr int TF_CTRL_REGS = 88, TF_SOFT_REGS = 208; // 128 * 88 + 256 * 208 <= 384 * 168
constexpr int TQ = 128, TK = 128;                    // rows of a query tile, keys of a key tile

struct alignas(64) TextMaps {
  CUtensorMap q, k, v;
};

template <int REGS> __device__ __forceinline__ void regs_up() { asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(REGS)); }
template <int REGS> __device__ __forceinline__ void regs_down() { asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(REGS)); }

template <int DH, bool BIAS>
__global__ void __launch_bounds__(TF_THREADS, 1)
text_fwd_kernel(const __grid_constant__ TextMaps maps, const __grid_constant__ MdbTextAttnArgs a, const int pair_heads) {
  constexpr int DBOX = DH / 64;               // 64-element (128 B) boxes along the head dimension
  constexpr int TILE_BYTES = TQ * DH * 2;
  constexpr int BOX_BYTES = TQ * 128;
  constexpr uint32_t S_COL0 = 0, S_COL1 = 128, O_COL0 = 256, O_COL1 = 384;

  extern __shared__ uint8_t smem_raw[];
  __shared__ uint64_t q_full, k_full[2], k_empty[2], v_full[2], v_empty[2];
  __shared__ uint64_t s_full[2], p_full[2][2], o_full[2];
  __shared__ uint32_t tmem_base_s;
  __shared__ int abort_s;

  const uint32_t raw_addr = smem_u32(smem_raw);
  uint8_t* smem = smem_raw + (((raw_addr + 1023u) & ~1023u) - raw_addr);
  uint8_t* sQ = smem;                       // 2 tiles
  uint8_t* sK = sQ + 2 * TILE_BYTES;        // 2 stages
  uint8_t* sV = sK + 2 * TILE_BYTES;        // 2 stages
  float* lut = reinterpret_cast<float*>(sV + 2 * TILE_BYTES);     // BIAS: log2(e) * bias of the distances -near - 254 .. near + 254

  const int warp = threadIdx.x >> 5;
  const int lane = threadIdx.x & 31;
  const int batch = blockIdx.z;
  // with a mask that grows along the prompt the last rows have the most keys: they start first
  const int block = BIAS ? blockIdx.x : gridDim.x - 1 - blockIdx.x;
  const int rep = a.H / a.Hkv;
  const int head0 = pair_heads ? 2 * blockIdx.y : blockIdx.y;
  const int kv_head = head0 / rep;
  const int q0_first = block * (pair_heads ? TQ : 2 * TQ);
  const auto tile_q0 = [&](int t) { return pair_heads ? q0_first : q0_first + t * TQ; };
  const auto tile_head = [&](int t) { return pair_heads ? head0 + t : head0; };

  // key tiles of either query tile, and of both together: [0, ns) and [lo, hi)
  const TextSight sight = text_sight(a, batch);
  TextKeys all = {0, 0, 0};
  int t_ns[2], t_lo[2], t_hi[2];
#pragma unroll
  for (int t = 0; t < 2; ++t) {
    const int q0 = tile_q0(t);
    TextKeys k = {0, 0, 0};
    if (q0 < a.Sq) k = text_keys<BIAS>(a, sight, sight.start + q0, sight.start + min(q0 + TQ, a.Sq) - 1);
    t_ns[t] = (k.sinks + TK - 1) / TK;
    t_lo[t] = k.lo / TK;
    t_hi[t] = k.end > k.lo ? (k.end + TK - 1) / TK : t_lo[t];
    if (t == 0) all = k;
    else if (k.end > 0) {
      // the second tile's rows stand behind the first one's: its windows reach further, and begin later
      if (all.end == 0) all = k;
      else all.end = max(all.end, k.end);
    }
  }
  const int ns = max(t_ns[0], t_ns[1]);
  const int lo = max(all.lo / TK, ns);
  const int hi = max(max(t_hi[0], t_hi[1]), lo);
  const int n_kv = ns + hi - lo;
  const auto key_tile = [&](int i) { return i < ns ? i : i - ns + lo; };
  const auto active = [&](int t, int i) {
    const int kt = key_tile(i);
    return i < n_kv && (kt < t_ns[t] || (kt >= t_lo[t] && kt < t_hi[t]));
  };

  if (threadIdx.x == 0) {
    mbar_init(&q_full, 1);
    for (int s = 0; s < 2; ++s) {
      mbar_init(&k_full[s], 1);
      mbar_init(&k_empty[s], 1);
      mbar_init(&v_full[s], 1);
      mbar_init(&v_empty[s], 1);
      mbar_init(&s_full[s], 1);
      mbar_init(&p_full[s][0], 4);
      mbar_init(&p_full[s][1], 4);
      mbar_init(&o_full[s], 1);
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
  const int near = BIAS ? text_near(a) : 0;
  if (BIAS) {
    for (int i = threadIdx.x; i < 2 * near + 509; i += TF_THREADS)
      lut[i] = TXT_LOG2E * text_param(a.table, a.param_f32, static_cast<long long>(text_bucket(a, i - near - 254)) * a.H + head0);
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem_base = tmem_base_s;

  if (warp < 4) {
    regs_down<TF_CTRL_REGS>();
    if (warp == 0 && n_kv > 0) {
      // ----------------------------- TMA producer -----------------------------
      if (elect_one()) {
        mbar_expect_tx(&q_full, 2 * TILE_BYTES);
        for (int t = 0; t < 2; ++t)
          for (int d = 0; d < DBOX; ++d)
            tma_load_4d(sQ + t * TILE_BYTES + d * BOX_BYTES, &maps.q, &q_full, d * 64, tile_q0(t), tile_head(t), batch);
      }
      __syncwarp();
      bool ok = true;
      uint64_t* last_bar = &q_full;
      uint32_t last_par = 0;
      for (int i = 0; ok && i < n_kv; ++i) {
        const int st = i & 1;
        const uint32_t par = (i >> 1) & 1;
        for (int kv = 0; kv < 2; ++kv) {
          uint64_t* empty = kv ? &v_empty[st] : &k_empty[st];
          uint64_t* full = kv ? &v_full[st] : &k_full[st];
          ok = __all_sync(0xffffffffu, mbar_wait(empty, par ^ 1u, &abort_s));
          if (!ok) {
            if (lane == 0) report_status(a.status, STATUS_TIMEOUT, 111 + kv, i);
            break;
          }
          if (elect_one()) {
            mbar_expect_tx(full, TILE_BYTES);
            for (int d = 0; d < DBOX; ++d)
              tma_load_4d((kv ? sV : sK) + st * TILE_BYTES + d * BOX_BYTES, kv ? &maps.v : &maps.k, full, d * 64, key_tile(i) * TK, kv_head, batch);
          }
          __syncwarp();
          last_bar = full;
          last_par = par;
        }
      }
      if (!ok) {
        const uint64_t t0 = globaltimer_ns();
        while (!mbar_try_wait(last_bar, last_par) && globaltimer_ns() - t0 < 5000000ull) {
        }
      }
    } else if (warp == 1 && n_kv > 0) {
      // ----------------------------- MMA issue --------------------------------
      constexpr uint32_t idesc_s = make_idesc(1, UMMA_BF16, UMMA_BF16, 0, 0, TQ, TK);
      constexpr uint32_t idesc_pv = make_idesc(1, UMMA_BF16, UMMA_BF16, 0, 1, TQ, DH);
      const uint32_t s_tmem[2] = {tmem_base + S_COL0, tmem_base + S_COL1};
      const uint32_t o_tmem[2] = {tmem_base + O_COL0, tmem_base + O_COL1};
      const uint64_t q_desc = make_desc_kmajor_sw128(smem_u32(sQ)), k_desc = make_desc_kmajor_sw128(smem_u32(sK));
      const uint64_t v_desc = make_desc_mnmajor_sw128(smem_u32(sV), BOX_BYTES);
      const auto issue_s = [&](int t, int st) {
#pragma unroll
        for (int kk = 0; kk < DH / 16; ++kk) {
          const uint32_t off = static_cast<uint32_t>((kk / 4) * BOX_BYTES + (kk % 4) * 32) >> 4;
          umma_f16_ss(s_tmem[t], q_desc + (t * TILE_BYTES >> 4) + off, k_desc + (st * TILE_BYTES >> 4) + off, idesc_s, kk != 0 ? 1u : 0u);
        }
        umma_commit(&s_full[t]);
      };
      const auto issue_pv = [&](int t, int st, int half, bool first) {
#pragma unroll
        for (int k2 = 0; k2 < TK / 32; ++k2) {
          const int kk = half * (TK / 32) + k2;
          umma_f16_ts(o_tmem[t], s_tmem[t] + kk * 8, v_desc + ((st * TILE_BYTES + kk * 2048) >> 4), idesc_pv, (first && kk == 0) ? 0u : 1u);
        }
      };
      int done[2] = {0, 0};                 // key tiles that either query tile has finished
      bool ok = __all_sync(0xffffffffu, mbar_wait(&q_full, 0, &abort_s) && mbar_wait(&k_full[0], 0, &abort_s));
      if (!ok && lane == 0) report_status(a.status, STATUS_TIMEOUT, 121, 0);
      if (ok) {
        tc_fence_after();
        if (elect_one()) {
          for (int t = 0; t < 2; ++t)
            if (active(t, 0)) issue_s(t, 0);
          umma_commit(&k_empty[0]);
        }
        __syncwarp();
      }
      for (int i = 0; ok && i < n_kv; ++i) {
        const int st = i & 1, st_n = st ^ 1;
        const bool more = i + 1 < n_kv;
        ok = __all_sync(0xffffffffu, mbar_wait(&v_full[st], (i >> 1) & 1, &abort_s) && (!more || mbar_wait(&k_full[st_n], ((i + 1) >> 1) & 1, &abort_s)));
        if (!ok) {
          if (lane == 0) report_status(a.status, STATUS_TIMEOUT, 122, i);
          break;
        }
        const int k0 = key_tile(i) * TK;
        if (k0 + TK > all.end || (k0 < all.lo && k0 + TK > all.sinks)) {
          for (int r = lane; r < TK; r += 32) {
            const int j = k0 + r;
            if (j < all.end && (j >= all.lo || j < all.sinks)) continue;
            for (int d = 0; d < DBOX; ++d)
              for (int c = 0; c < 8; ++c)
                *reinterpret_cast<uint4*>(sV + st * TILE_BYTES + d * BOX_BYTES + r * 128 + ((c + r) & 7) * 16) = make_uint4(0, 0, 0, 0);
          }
          fence_proxy_async_smem();
          __syncwarp();
        }
        for (int t = 0; ok && t < 2; ++t) {
          const bool mine = active(t, i);
          for (int half = 0; ok && mine && half < 2; ++half) {
            ok = __all_sync(0xffffffffu, mbar_wait(&p_full[t][half], done[t] & 1, &abort_s));
            if (!ok) {
              if (lane == 0) report_status(a.status, STATUS_TIMEOUT, 123 + t, i);
              break;
            }
            tc_fence_after();
            if (elect_one()) {
              issue_pv(t, st, half, done[t] == 0);
              if (half == 1) umma_commit(&o_full[t]);
            }
            __syncwarp();
          }
          if (!ok) break;
          done[t] += mine;
          if (elect_one()) {
            if (more && active(t, i + 1)) issue_s(t, st_n);
            if (t == 1) {
              umma_commit(&v_empty[st]);
              if (more) umma_commit(&k_empty[st_n]);
            }
          }
          __syncwarp();
        }
      }
    }
    __syncwarp();
  } else {
    // ------------------------------- softmax: one thread per query row -----------------------
    regs_up<TF_SOFT_REGS>();
    const int t = (warp - 4) >> 2;
    const int quad = warp & 3;
    const uint32_t lane_addr = static_cast<uint32_t>(quad * 32) << 16;
    const uint32_t s_tile = tmem_base + lane_addr + (t ? S_COL1 : S_COL0);
    const uint32_t o_addr = tmem_base + lane_addr + (t ? O_COL1 : O_COL0);
    const int q0 = tile_q0(t), head = tile_head(t);
    const int row = q0 + quad * 32 + lane;
    const int p = sight.start + row, p_first = sight.start + q0, p_last = p_first + TQ - 1;
    const float sl2 = a.scale * TXT_LOG2E;
    const float far_before = BIAS ? lut[0] : 0.f, far_behind = BIAS ? lut[2 * near + 508] : 0.f;
    // The reference m and the divisor l; a sink logit is the first member of the sum.
    float m_used = -INFINITY, l_run[2] = {0.f, 0.f};
    if (!BIAS && a.sink_logits != nullptr) {
      m_used = TXT_LOG2E * text_param(a.sink_logits, a.param_f32, head);
      l_run[0] = m_used == -INFINITY ? 0.f : 1.f;
    }
    bool ok = true;
    int done = 0;

    for (int i = 0; ok && i < n_kv; ++i) {
      if (!active(t, i)) continue;
      const int k0 = key_tile(i) * TK;
      ok = __all_sync(0xffffffffu, mbar_wait(&s_full[t], done & 1, &abort_s));
      if (!ok) {
        if (lane == 0) report_status(a.status, STATUS_TIMEOUT, 131 + t, i);
        break;
      }
      tc_fence_after();
      uint32_t sv[4][32];
#pragma unroll
      for (int c = 0; c < 4; ++c) tmem_ld_32x32b_x32(s_tile + c * 32, sv[c]);
      tmem_wait_ld();
      float mul = sl2, add = 0.f;           // exponent = mul * score + add - m
      if (BIAS) {
        const int d = k0 - q0;
        if (d - 127 >= near) add = far_behind;
        else if (d + 127 <= -near) add = far_before;
        else {
          const float* b = lut + near + 254 + k0 - row;
          mul = 1.f;
#pragma unroll
          for (int c = 0; c < 4; ++c)
#pragma unroll
            for (int e = 0; e < 32; ++e) sv[c][e] = __float_as_uint(fmaf(__uint_as_float(sv[c][e]), sl2, b[c * 32 + e]));
        }
        if (k0 + TK > sight.valid) {
#pragma unroll
          for (int c = 0; c < 4; ++c)
#pragma unroll
            for (int e = 0; e < 32; ++e)
              if (k0 + c * 32 + e >= sight.valid) sv[c][e] = 0xff800000u;        // -inf
        }
      } else if (!(k0 + TK - 1 <= p_first && k0 + TK <= sight.valid && (k0 > p_last - a.window || k0 + TK <= a.sinks))) {
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          const uint32_t see = text_mask(a, sight.valid, p, k0 + c * 32);
#pragma unroll
          for (int e = 0; e < 32; ++e)
            if (!(see >> e & 1u)) sv[c][e] = 0xff800000u;
        }
      }
      float mc[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
      for (int e = 0; e < 32; e += 2)
#pragma unroll
        for (int c = 0; c < 4; ++c) mc[c] = fmax3(mc[c], __uint_as_float(sv[c][e]), __uint_as_float(sv[c][e + 1]));
      const float mx = fmaf(fmaxf(fmaxf(mc[0], mc[1]), fmaxf(mc[2], mc[3])), mul, add);
      if (done == 0) {
        if (mx > m_used) {
          l_run[0] *= exp2f(m_used - mx);
          m_used = mx;
        }
      } else {
        // The reference is raised when a row has outgrown it by more than 2^8, and with the first key that a row sees.
        const bool need = mx > m_used + 8.0f;
        if (__any_sync(0xffffffffu, need)) {
          ok = __all_sync(0xffffffffu, mbar_wait(&o_full[t], (done - 1) & 1, &abort_s));
          if (!ok) {
            if (lane == 0) report_status(a.status, STATUS_TIMEOUT, 133 + t, i);
            break;
          }
          tc_fence_after();
          const float alpha = need ? exp2f(m_used - mx) : 1.0f;
          if (need) m_used = mx;
          l_run[0] *= alpha;
          l_run[1] *= alpha;
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
      float2 sum_a = make_float2(0.f, 0.f), sum_b = make_float2(0.f, 0.f);
      const float nm = add - (m_used == -INFINITY ? 0.f : m_used);          // no key so far: every exponent is -inf
      const float2 mul2 = make_float2(mul, mul), nm2 = make_float2(nm, nm);
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        uint32_t pk[16];
#pragma unroll
        for (int e = 0; e < 32; e += 4) {
          // half of every second group of four exponentials runs on the FMA pipe: the special-function unit bounds the rest
          const float2 x01 = ffma2(make_float2(__uint_as_float(sv[c][e]), __uint_as_float(sv[c][e + 1])), mul2, nm2);
          const float2 x23 = ffma2(make_float2(__uint_as_float(sv[c][e + 2]), __uint_as_float(sv[c][e + 3])), mul2, nm2);
          const float2 u = make_float2(ex2_approx(x01.x), ex2_approx(x23.x));
          float2 w;
          if ((e >> 2) % 2 == 1) w = ex2_poly2(make_float2(x01.y, x23.y), -127.f);
          else w = make_float2(ex2_approx(x01.y), ex2_approx(x23.y));
          sum_a = fadd2(sum_a, u);
          sum_b = fadd2(sum_b, w);
          pk[e >> 1] = pack_bf16x2(u.x, w.x);
          pk[(e >> 1) + 1] = pack_bf16x2(u.y, w.y);
        }
        tmem_st_32x32b_x16(s_tile + c * 16, pk);          // over scores that are in registers by now
        if (c & 1) {
          tmem_wait_st();
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(&p_full[t][c >> 1]);
          l_run[c >> 1] += (sum_a.x + sum_a.y) + (sum_b.x + sum_b.y);
          sum_a = sum_b = make_float2(0.f, 0.f);
        }
      }
      ++done;
    }
    if (ok && done > 0) {
      ok = __all_sync(0xffffffffu, mbar_wait(&o_full[t], (done - 1) & 1, &abort_s));
      if (!ok && lane == 0) report_status(a.status, STATUS_TIMEOUT, 135 + t, n_kv);
    }
    if (ok) {
      tc_fence_after();
      const bool empty = done == 0 || m_used == -INFINITY;
      const float l_tot = l_run[0] + l_run[1];
      const float inv_l = 1.f / l_tot;
      // Whole rows leave through the tile's Q buffer (its products have completed): DH / 8 lanes x 16 bytes a row. A tile without keys
      // has not waited for its Q and stores zeros from registers.
      constexpr int CH = DH / 8;
      uint8_t* stage = sQ + t * TILE_BYTES + quad * (32 * DH * 2);
      if (done > 0) {
        uint4* my_row = reinterpret_cast<uint4*>(stage + lane * (DH * 2));
#pragma unroll
        for (int c = 0; c < DH / 32; ++c) {
          uint32_t r[32];
          tmem_ld_32x32b_x32(o_addr + c * 32, r);
          tmem_wait_ld();
#pragma unroll
          for (int e = 0; e < 32; e += 8) {
            uint4 w;
            w.x = pack_bf16x2(__uint_as_float(r[e + 0]) * inv_l, __uint_as_float(r[e + 1]) * inv_l);
            w.y = pack_bf16x2(__uint_as_float(r[e + 2]) * inv_l, __uint_as_float(r[e + 3]) * inv_l);
            w.z = pack_bf16x2(__uint_as_float(r[e + 4]) * inv_l, __uint_as_float(r[e + 5]) * inv_l);
            w.w = pack_bf16x2(__uint_as_float(r[e + 6]) * inv_l, __uint_as_float(r[e + 7]) * inv_l);
            if (empty) w = make_uint4(0, 0, 0, 0);
            my_row[(c * 4 + (e >> 3)) ^ (lane & (CH - 1))] = w;
          }
        }
        __syncwarp();
      }
      const int chunk = lane % CH;
      __nv_bfloat16* o = static_cast<__nv_bfloat16*>(a.o) + batch * a.o_strides[0] + head * a.o_strides[2] + chunk * 8;
#pragma unroll 4
      for (int n = 0; n < CH; ++n) {
        const int rl = n * (32 / CH) + lane / CH;
        const int r = q0 + quad * 32 + rl;
        if (r >= a.Sq) continue;
        uint4 w = make_uint4(0, 0, 0, 0);
        if (done > 0) w = reinterpret_cast<const uint4*>(stage + rl * (DH * 2))[chunk ^ (rl & (CH - 1))];
        *reinterpret_cast<uint4*>(o + r * a.o_strides[1]) = w;
      }
      // +inf where a row saw nothing: the backward pass then finds probabilities of zero
      if (a.lse != nullptr && row < a.Sq)
        a.lse[(static_cast<long long>(batch) * a.H + head) * a.Sq + row] = l_tot > 0.f && m_used != -INFINITY ? m_used + log2f(l_tot) : INFINITY;
    }
  }

  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem_base, 512);
  }
}

static int text_map(CUtensorMap* m, const void* ptr, int B, int S, int H, int Dh, const long long* strides) {
  int64_t ext[4] = {Dh, S, H, B};
  int64_t str[4] = {2, strides[1] * 2, strides[2] * 2, strides[0] * 2};
  int box[4] = {64, 128, 1, 1};
  return mdb_make_tmap(m, ptr, 2, 4, ext, str, box, 1);
}

template <int DH, bool BIAS>
static int launch_text_fwd(const TextMaps& maps, const MdbTextAttnArgs& a, cudaStream_t st) {
  constexpr int MOST = 6 * TQ * DH * 2 + 1024 + (BIAS ? (2 * MDB_TEXT_MAX_DISTANCE + 509) * 4 : 0);
  auto kern = text_fwd_kernel<DH, BIAS>;
  static bool ready[TXT_DEVICES];
  if (int r = allow_smem(kern, MOST, ready)) return r;
  const int smem = 6 * TQ * DH * 2 + 1024 + (BIAS ? (2 * text_near(a) + 509) * 4 : 0);
  // Two heads of a group on the same rows read the same key tiles, whatever the window; two row blocks would also visit each other's.
  // The bias table in shared memory is one head's.
  const int pair_heads = !BIAS && (a.H / a.Hkv) % 2 == 0;
  const int rows = pair_heads ? TQ : 2 * TQ;
  kern<<<dim3((a.Sq + rows - 1) / rows, pair_heads ? a.H / 2 : a.H, a.B), TF_THREADS, smem, st>>>(maps, a, pair_heads);
  return static_cast<int>(cudaGetLastError());
}

int text_attention_prompt(const MdbTextAttnArgs& a, cudaStream_t st) {
  TextMaps maps;
  int r = text_map(&maps.q, a.q, a.B, a.Sq, a.H, a.Dh, a.q_strides);
  if (r) return 1000 + r;
  r = text_map(&maps.k, a.k, a.B, a.Skv, a.Hkv, a.Dh, a.k_strides);
  if (r) return 2000 + r;
  r = text_map(&maps.v, a.v, a.B, a.Skv, a.Hkv, a.Dh, a.v_strides);
  if (r) return 3000 + r;
  if (a.table != nullptr) return a.Dh == 128 ? launch_text_fwd<128, true>(maps, a, st) : launch_text_fwd<64, true>(maps, a, st);
  return a.Dh == 128 ? launch_text_fwd<128, false>(maps, a, st) : launch_text_fwd<64, false>(maps, a, st);
}

}  // namespace mdb

MDB_DEFINE_WAIT_LIMIT_SETTER(mdb_set_wait_limit_text_fwd)
