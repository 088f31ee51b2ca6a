// The language models' attention for a few tokens over a cache (decoding, drafted tokens): at most 64 rows per key head, a row being one query of
// one head of the group, and more keys than queries. No log-sum-exp is kept.
//
//   o_i = sum_j exp2(x_ij - M_i) v_j / sum_j exp2(x_ij - M_i): every warp forms the sums over its keys with its own reference m, and the parts are
//   joined with the factors exp2(m - M).
//
// Keys and values are read once and bound the time, so the split is over keys: the CTAs of a cluster share the keys of one key head of one
// sequence, the four warps of a CTA the 64 keys of a stage (with more than 16 rows fewer keys and 16 rows each). Stages arrive by TMA, started by a warp of
// their own. Products are mma.sync m16n8k16: 16 rows are all there is to multiply, a 128-row tcgen05 tile would be mostly padding. A
// probability goes into its product as two bf16 terms, so only the output is rounded; the memory leaves time for the second product.
// The warps' parts meet in shared memory, the CTAs' in the cluster's distributed shared memory: one launch, no workspace.
//
// Visited are the tiles of the first `sinks` keys and those from the oldest key of a window on, wherever that is. Rows of V that no query sees
// are zeroed in shared memory before the product (0 * NaN is not 0).
//
// 4 sequences of 70001 to 131072 keys, 8 key heads of 128: 256 to 276 us, 6.1 to 6.4 TB/s of keys and values, which the memory bounds. 16 of 1 to 16384 keys
// with window 4096 and 4 first keys: 41 to 45 us for 213 to 263 MB, 5.2 to 5.8 TB/s; every sequence has the same two CTAs per key head, so that short ones
// leave their part of the memory's rate unused. The smallest calls are one launch of 5 us.
#include "text_attention.cuh"
#include "gemm_api.h"

#include <algorithm>
#include <string.h>

namespace mdb {

constexpr int SK = 64;                      // keys of a stage
constexpr int STEP_WARPS = 4, STEP_THREADS = (STEP_WARPS + 1) * 32;

struct alignas(64) StepMaps {
  CUtensorMap k, v;
};

__device__ __forceinline__ void ldsm_x4(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ void ldsm_x4_t(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ void mma_bf16(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
               : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
               : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
template <int DH> struct StepShape {
  static constexpr int TILE = SK * DH * 2;                  // K or V of a stage
  static constexpr int STAGES = DH == 128 ? 3 : 6;          // 96 KB, so that two CTAs share an SM and 192 KB are on the way
  static constexpr int BYTES = STAGES * 2 * TILE + 1024;
};

// MT: tiles of 16 rows
template <int DH, int MT>
__global__ void __launch_bounds__(STEP_THREADS)
text_step_kernel(const __grid_constant__ StepMaps maps, const __grid_constant__ MdbTextAttnArgs a) {
  using Shape = StepShape<DH>;
  constexpr int TILE = Shape::TILE, STAGES = Shape::STAGES, BOX = SK * 128;
  constexpr int ROWS = 16 * MT, PER_TILE = STEP_WARPS / MT;           // warps that share the keys of a stage
  constexpr int WK = SK / PER_TILE;                                   // keys of a warp in a stage

  extern __shared__ uint8_t smem_raw[];
  __shared__ uint64_t full[STAGES], empty[STAGES];
  __shared__ int abort_s;
  __shared__ float part_m[STEP_WARPS][16], part_l[STEP_WARPS][16];
  __shared__ float cta_m[ROWS], cta_l[ROWS];
  uint8_t* smem = smem_raw + (((smem_u32(smem_raw) + 1023u) & ~1023u) - smem_u32(smem_raw));

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int ranks = gridDim.x, rank = blockIdx.x;                     // the grid's x extent is one cluster
  const int kv_head = blockIdx.y, batch = blockIdx.z;
  const int rep = a.H / a.Hkv, rows = rep * a.Sq;

  const TextSight sight = text_sight(a, batch);
  const TextKeys keys = text_keys<false>(a, sight, sight.start, sight.start + a.Sq - 1);
  const int ns = (keys.sinks + SK - 1) / SK;
  const int lo = max(keys.lo, keys.sinks);
  const int n_all = ns + (max(keys.end - lo, 0) + SK - 1) / SK;
  const int first = static_cast<int>(static_cast<long long>(n_all) * rank / ranks), n = static_cast<int>(static_cast<long long>(n_all) * (rank + 1) / ranks) - first;
  const auto tile_key = [&](int i) { return first + i < ns ? (first + i) * SK : lo + (first + i - ns) * SK; };
  // keys of tile i end here: the first ones do not run into the windows, which begin with a tile of their own
  const auto tile_end = [&](int i) { return first + i < ns ? keys.sinks : keys.end; };

  if (threadIdx.x == 0) {
    for (int s = 0; s < STAGES; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], STEP_WARPS);
    }
    abort_s = 0;
    fence_mbar_init();
  }
  __syncthreads();

  float o[DH / 8][4];
#pragma unroll
  for (int d = 0; d < DH / 8; ++d)
#pragma unroll
    for (int e = 0; e < 4; ++e) o[d][e] = 0.f;
  float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f};             // of the rows lane / 4 and lane / 4 + 8 of the warp's tile

  if (warp == STEP_WARPS) {
    if (lane == 0) {
      bool ok = true;
      int i = 0;
      for (; i < n; ++i) {
        const int st = i % STAGES;
        ok = mbar_wait(&empty[st], ((i / STAGES) & 1) ^ 1u, &abort_s);
        if (!ok) {
          report_status(a.status, STATUS_TIMEOUT, 171, i);
          break;
        }
        mbar_expect_tx(&full[st], 2 * TILE);
        for (int d = 0; d < DH / 64; ++d) {
          tma_load_4d(smem + st * 2 * TILE + d * BOX, &maps.k, &full[st], d * 64, tile_key(i), kv_head, batch);
          tma_load_4d(smem + st * 2 * TILE + TILE + d * BOX, &maps.v, &full[st], d * 64, tile_key(i), kv_head, batch);
        }
      }
      if (!ok) {      // the copies on the way land before the memory is used for anything else
        for (int j = max(0, i - STAGES); j < i; ++j) {
          const uint64_t t0 = globaltimer_ns();
          while (!mbar_try_wait(&full[j % STAGES], (j / STAGES) & 1) && globaltimer_ns() - t0 < 5000000ull) {
          }
        }
      }
    }
    __syncwarp();
  } else {
    const int mt = warp / PER_TILE, part = warp % PER_TILE;
    const int r_lo = mt * 16 + (lane >> 2);                           // rows r_lo and r_lo + 8, columns from 2 * (lane % 4)
    uint32_t q[DH / 16][4];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int r = r_lo + 8 * h;
      const __nv_bfloat16* p = static_cast<const __nv_bfloat16*>(a.q) + batch * a.q_strides[0] + (r / rep) * a.q_strides[1] +
                               (kv_head * rep + r % rep) * a.q_strides[2] + 2 * (lane & 3);
#pragma unroll
      for (int kk = 0; kk < DH / 16; ++kk) {
        q[kk][h] = r < rows ? *reinterpret_cast<const uint32_t*>(p + kk * 16) : 0u;
        q[kk][h + 2] = r < rows ? *reinterpret_cast<const uint32_t*>(p + kk * 16 + 8) : 0u;
      }
    }
    const float sl2 = a.scale * TXT_LOG2E;
    const int p_row[2] = {sight.start + r_lo / rep, sight.start + (r_lo + 8) / rep};
    const int p_last = sight.start + a.Sq - 1;
    bool ok = true;
    for (int i = 0; i < n; ++i) {
      const int st = i % STAGES;
      ok = __all_sync(0xffffffffu, mbar_wait(&full[st], (i / STAGES) & 1, &abort_s));
      if (!ok) {
        if (lane == 0) report_status(a.status, STATUS_TIMEOUT, 172, i);
        break;
      }
      const uint8_t* sk = smem + st * 2 * TILE;
      uint8_t* sv = smem + st * 2 * TILE + TILE;
      const int k0 = tile_key(i) + part * WK, k_end = tile_end(i);
      if (k0 + WK > k_end) {
        for (int r = lane; r < WK; r += 32)
          if (k0 + r >= k_end)
            for (int b = 0; b < DH / 64; ++b)
              for (int c = 0; c < 8; ++c) *reinterpret_cast<uint4*>(sv + b * BOX + (part * WK + r) * 128 + ((c + r) & 7) * 16) = make_uint4(0, 0, 0, 0);
        __syncwarp();
        fence_proxy_async_smem();
      }
#pragma unroll
      for (int s16 = 0; s16 < WK / 16; ++s16) {
        const int kr = part * WK + s16 * 16, kb = k0 + s16 * 16;      // row in the stage, key
        if (kb >= k_end) break;
        float x[2][4];
#pragma unroll
        for (int nt = 0; nt < 2; ++nt) {
#pragma unroll
          for (int e = 0; e < 4; ++e) x[nt][e] = 0.f;
          const int r = kr + nt * 8 + (lane & 7);
#pragma unroll
          for (int kk = 0; kk < DH / 16; kk += 2) {
            uint32_t b[4];
            const int c = (kk & 3) * 2 + (lane >> 3);                 // 16-byte piece of the row's 128 bytes
            ldsm_x4(b, smem_u32(sk) + (kk >> 2) * BOX + r * 128 + ((c ^ (r & 7)) << 4));
            mma_bf16(x[nt], q[kk], b[0], b[1]);
            mma_bf16(x[nt], q[kk + 1], b[2], b[3]);
          }
        }
        // visible whole: behind no query's position, inside every window, before the end
        const bool whole = kb + 15 <= sight.start && kb + 16 <= k_end && (kb > p_last - a.window || kb + 16 <= a.sinks);
#pragma unroll
        for (int nt = 0; nt < 2; ++nt)
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            x[nt][e] *= sl2;
            if (!whole) {
              const int j = kb + nt * 8 + 2 * (lane & 3) + (e & 1), p = p_row[e >> 1];
              if (!(j <= p && j < k_end && (p - j < a.window || j < a.sinks))) x[nt][e] = -INFINITY;
            }
          }
        float f[2];
        bool raise = false;
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          float t = max_nan(max3_nan(x[0][2 * h], x[0][2 * h + 1], x[1][2 * h]), x[1][2 * h + 1]);
          t = max_nan(t, __shfl_xor_sync(0xffffffffu, t, 1));
          t = max_nan(t, __shfl_xor_sync(0xffffffffu, t, 2));
          // the reference is raised when outgrown by more than 2^8, and with the first key that the row sees; NaN is kept
          f[h] = 1.f;
          if (!(t <= m[h] + 8.f)) {
            f[h] = exp2f(m[h] - t);
            m[h] = max_nan(m[h], t);
            raise = true;
          }
        }
        if (__any_sync(0xffffffffu, raise)) {
          l[0] *= f[0];
          l[1] *= f[1];
#pragma unroll
          for (int d = 0; d < DH / 8; ++d) {
            o[d][0] *= f[0];
            o[d][1] *= f[0];
            o[d][2] *= f[1];
            o[d][3] *= f[1];
          }
        }
        uint32_t ph[4], pl[4];
#pragma unroll
        for (int nt = 0; nt < 2; ++nt)
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const float mr = m[h] == -INFINITY ? 0.f : m[h];
            const float p0 = ex2_approx(x[nt][2 * h] - mr), p1 = ex2_approx(x[nt][2 * h + 1] - mr);
            l[h] += p0 + p1;
            ph[nt * 2 + h] = pack_bf16x2(p0, p1);
            const float2 back = unpack_bf16x2(ph[nt * 2 + h]);
            pl[nt * 2 + h] = pack_bf16x2(p0 - back.x, p1 - back.y);
          }
#pragma unroll
        for (int d = 0; d < DH / 8; d += 2) {
          uint32_t b[4];
          const int r = kr + (lane & 15), c = (d & 7) + (lane >> 4);
          ldsm_x4_t(b, smem_u32(sv) + (d >> 3) * BOX + r * 128 + ((c ^ (r & 7)) << 4));
          mma_bf16(o[d], ph, b[0], b[1]);
          mma_bf16(o[d + 1], ph, b[2], b[3]);
          mma_bf16(o[d], pl, b[0], b[1]);
          mma_bf16(o[d + 1], pl, b[2], b[3]);
        }
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(&empty[st]);
    }
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      l[h] += __shfl_xor_sync(0xffffffffu, l[h], 1);
      l[h] += __shfl_xor_sync(0xffffffffu, l[h], 2);
      if ((lane & 3) == 0) {
        part_m[warp][(lane >> 2) + 8 * h] = m[h];
        part_l[warp][(lane >> 2) + 8 * h] = l[h];
      }
    }
  }
  // the stages' memory is free: [warp][16][DH] parts, then [ROWS][DH] of the CTA
  __syncthreads();
  float* slab = reinterpret_cast<float*>(smem);
  float* whole_o = slab + STEP_WARPS * 16 * DH;
  if (warp < STEP_WARPS) {
    float* mine = slab + warp * 16 * DH + (lane >> 2) * DH + 2 * (lane & 3);
#pragma unroll
    for (int d = 0; d < DH / 8; ++d) {
      *reinterpret_cast<float2*>(mine + d * 8) = make_float2(o[d][0], o[d][1]);
      *reinterpret_cast<float2*>(mine + 8 * DH + d * 8) = make_float2(o[d][2], o[d][3]);
    }
  }
  __syncthreads();
  for (int e = threadIdx.x; e < ROWS * DH / 4; e += STEP_THREADS) {
    const int r = e / (DH / 4), w0 = (r / 16) * PER_TILE, rr = r % 16, c = e % (DH / 4) * 4;
    float top = part_m[w0][rr];
#pragma unroll
    for (int w = 1; w < PER_TILE; ++w) top = max_nan(top, part_m[w0 + w][rr]);
    float4 s = make_float4(0.f, 0.f, 0.f, 0.f);
    float sum = 0.f;
#pragma unroll
    for (int w = 0; w < PER_TILE; ++w) {
      const float f = part_m[w0 + w][rr] == -INFINITY ? 0.f : exp2f(part_m[w0 + w][rr] - top);
      const float4 v = *reinterpret_cast<const float4*>(slab + (w0 + w) * 16 * DH + rr * DH + c);
      s.x += f * v.x;
      s.y += f * v.y;
      s.z += f * v.z;
      s.w += f * v.w;
      sum += f * part_l[w0 + w][rr];
    }
    *reinterpret_cast<float4*>(whole_o + r * DH + c) = s;
    if (c == 0) {
      cta_m[r] = top;
      cta_l[r] = sum;
    }
  }
  __syncthreads();
  if (ranks > 1) {
    __syncwarp();
    cluster_arrive();
    cluster_wait();
  }
  // every CTA of the cluster joins and stores a share of the elements
  for (int e = threadIdx.x + rank * STEP_THREADS; e < rows * DH / 4; e += ranks * STEP_THREADS) {
    const int r = e / (DH / 4), c = e % (DH / 4) * 4;
    const int h = kv_head * rep + r % rep;
    float top = -INFINITY, sum = 0.f;
    if (a.sink_logits != nullptr) {
      top = TXT_LOG2E * text_param(a.sink_logits, a.param_f32, h);
      sum = top == -INFINITY ? 0.f : 1.f;
    }
    float4 s = make_float4(0.f, 0.f, 0.f, 0.f);
    for (int k = 0; k < ranks; ++k) {
      const float mk = ranks > 1 ? ld_cluster_f32(mapa_shared(smem_u32(&cta_m[r]), k)) : cta_m[r];
      if (mk == -INFINITY) continue;
      const float lk = ranks > 1 ? ld_cluster_f32(mapa_shared(smem_u32(&cta_l[r]), k)) : cta_l[r];
      const float4 v = ranks > 1 ? ld_cluster_f32x4(mapa_shared(smem_u32(whole_o + r * DH + c), k)) : *reinterpret_cast<const float4*>(whole_o + r * DH + c);
      const float up = fmaxf(top, mk), f = exp2f(top - up), g = exp2f(mk - up);
      s.x = s.x * f + v.x * g;
      s.y = s.y * f + v.y * g;
      s.z = s.z * f + v.z * g;
      s.w = s.w * f + v.w * g;
      sum = sum * f + lk * g;
      top = up;
    }
    const float inv = sum > 0.f ? 1.f / sum : 0.f;
    uint2 w;
    w.x = pack_bf16x2(s.x * inv, s.y * inv);
    w.y = pack_bf16x2(s.z * inv, s.w * inv);
    *reinterpret_cast<uint2*>(static_cast<__nv_bfloat16*>(a.o) + batch * a.o_strides[0] + (r / rep) * a.o_strides[1] + h * a.o_strides[2] + c) = w;
  }
  if (ranks > 1) {      // no CTA leaves while another one reads its part
    __syncwarp();
    cluster_arrive();
    cluster_wait();
  }
}

template <int DH, int MT>
static int launch_step(const StepMaps& maps, const MdbTextAttnArgs& a, int ranks, cudaStream_t st) {
  auto kern = text_step_kernel<DH, MT>;
  static bool ready[TXT_DEVICES], wide[TXT_DEVICES];
  if (int r = allow_smem(kern, StepShape<DH>::BYTES, ready)) return r;
  if (int r = allow_wide_clusters(kern, wide)) return r;
  cudaLaunchConfig_t c;
  memset(&c, 0, sizeof(c));
  c.gridDim = dim3(ranks, a.Hkv, a.B);
  c.blockDim = dim3(STEP_THREADS);
  c.dynamicSmemBytes = StepShape<DH>::BYTES;
  c.stream = st;
  cudaLaunchAttribute at;
  at.id = cudaLaunchAttributeClusterDimension;
  at.val.clusterDim.x = ranks;
  at.val.clusterDim.y = at.val.clusterDim.z = 1;
  c.attrs = &at;
  c.numAttrs = 1;
  return static_cast<int>(cudaLaunchKernelEx(&c, kern, maps, a));
}

static int step_map(CUtensorMap* m, const void* ptr, const MdbTextAttnArgs& a, const long long* strides) {
  int64_t ext[4] = {a.Dh, a.Skv, a.Hkv, a.B};
  int64_t str[4] = {2, strides[1] * 2, strides[2] * 2, strides[0] * 2};
  int box[4] = {64, SK, 1, 1};
  return mdb_make_tmap(m, ptr, 2, 4, ext, str, box, 1);
}

// Few rows over more keys than their own. A whole prompt goes to the other kernel however short it is, so that a token's result has the same bits whatever the
// length that its prompt is padded to. Device times in us with 8 / 16 / 32 / 64 rows, and of the other kernel: 32 / 8 heads of 128, one sequence of 8192
// keys 18 / 19 / 25 / 39, 109; 64 of 1100 keys 55 / 57 / 75 / 135, 142 to 145; 32 of 16384 with window 4096 84 / 85 / 121 / 225, 265; 64 / 8 heads of 64, one of
// 8192 15 / 16 / 21 / 31, 117. Only 64 rows over 300 keys are slower here: 17 us, 11.5.
bool text_attention_is_step(const MdbTextAttnArgs& a) {
  return a.lse == nullptr && a.table == nullptr && a.Skv > a.Sq && static_cast<long long>(a.Sq) * (a.H / a.Hkv) <= 64;
}

int text_attention_step(const MdbTextAttnArgs& a, cudaStream_t st) {
  StepMaps maps;
  int r = step_map(&maps.k, a.k, a, a.k_strides);
  if (r) return 2000 + r;
  r = step_map(&maps.v, a.v, a, a.v_strides);
  if (r) return 3000 + r;
  // A cluster has as many CTAs as give each two stages or more of the longest key range, up to sixteen, while the SMs hold them all at two each.
  // One sequence, with 8 / 16 CTAs: 8000 keys of 8 heads of 128 19.8 / 17.4 us, 32000 keys of 4 heads 57.9 / 35.2.
  const long long most = std::min<long long>(a.Skv, static_cast<long long>(a.window) + a.sinks + a.Sq - 1);
  const long long stages = (most + SK - 1) / SK, groups = static_cast<long long>(a.B) * a.Hkv;
  int ranks = 1;
  while (ranks < 16 && 4 * ranks <= stages && groups * ranks * 2 <= 2 * device_sm_count()) ranks *= 2;
  const int rows = a.Sq * (a.H / a.Hkv);
  if (a.Dh == 128) {
    if (rows <= 16) return launch_step<128, 1>(maps, a, ranks, st);
    return rows <= 32 ? launch_step<128, 2>(maps, a, ranks, st) : launch_step<128, 4>(maps, a, ranks, st);
  }
  if (rows <= 16) return launch_step<64, 1>(maps, a, ranks, st);
  return rows <= 32 ? launch_step<64, 2>(maps, a, ranks, st) : launch_step<64, 4>(maps, a, ranks, st);
}

}  // namespace mdb

MDB_DEFINE_WAIT_LIMIT_SETTER(mdb_set_wait_limit_text_step)
