// Attention over the pages of several sequences: query row i of sequence b stands at position p = kv_len[b] - Sq + i and sees the keys up to p.
//
//   o_i = sum_j p_ij v_j / sum_j p_ij,  p_ij = exp2(x_ij - m_i),  x_ij = log2(e) scale 2^ek q_i . k_j;  values are in units of 2^ev; ek, ev of the page and head
//
// A few queries (at most 64 rows per key head, a row being one query of one head of the group): keys and values are read once and bound the time, so the work is split
// over keys. All tiles of 128 keys of all sequences and key heads are one line, of which every CTA takes an equal part, wherever that begins and ends: sequences of 1 and
// of 100000 tokens share the memory's rate. A CTA's tiles of one sequence and head ("segment") end in an output, or in a part (m, l, o) where other CTAs have tiles of
// it too; a second, small kernel joins those in order. It is launched with the first one and waits for its end. Where no sequence has more than four tiles, a CTA takes one
// sequence and head each instead, and there is nothing to join.
//
// A warp of its own starts the copies: it knows the pages of the next 32 places of the table and their scales, and brings K and V of a tile in by TMA, one box
// per page. Four or eight warps multiply, with mma.sync m16n8k16: S^T = K Q^T and O^T = V^T P^T, so that the keys and the columns of V fill the 16 and the rows, of which there
// are few, the 8. (A 128-row tcgen05 tile would be mostly padding.) Each warp has 32 keys at a time; where a warp has no room for all rows the warps share out those.
//
// 8 bits: e4m3 values are exact in f16, and two of them take one conversion, so the products are f16 ones. Of a key's row a lane reads 16 bytes as they lie; which
// of them are columns 2t, 2t + 1 of a k-step is free as long as the queries' registers use the same order, and so no byte is moved. For values ldmatrix transposes pairs of bytes,
// and one byte permutation makes two columns of them. Queries are brought to [1, 2) by a power of two per row, which leaves them exact but for those below 2^-14 of
// the row's largest (2^-25 of it at most). A value's power of two goes into its probability: the product is of w_ij = p_ij 2^(ev - u_i), rounded to f16 (2^-11, where the output's
// rounding is 2^-8). The reference m_i is kept 2^7 below the first maximum of x_ij, and the whole number u_i follows so that the largest w_ij is between about 2^6 and 2^15: whatever the
// pages' units are, weights down to 2^-20 of the largest have all their bits (with one u for all rows, the largest unit met, a page that a row hardly sees took the bits of those that it sees).
// bf16: the products are bf16 ones; a probability goes into its product as two bf16 terms, so only the output is rounded.
//
// Keys behind the sequence's end are masked and their values zeroed in shared memory before the product (0 * NaN is not 0).
//
// What bounds it: memory where sequences are long. 4 tokens over 70001 to 131072 positions, 32 / 8 heads of 128, e4m3: 129 us, 5.95 TB/s (0.91 of the measured rate; bf16, 16 over 16384: 182 us, 5.9 TB/s). 32 over 0 to 16384:
// 82 us, 4.4 TB/s: 12000 cycles to a CTA's first tile (lengths, table, scales and data one after the other), then 3200 a tile of which it works 1300. Few rows leave latencies: one token over 300
// positions 7 us on the device. With more than 16 rows the turns of a warp: 40 rows over bf16 pages, heads of 64, 5600 cycles a tile of 128 keys, 27 us for 8 sequences of 17 to 4091; 32 rows over 8 bits, heads of 128,
// 8 sequences of 4000, 46 us.
// Keys as the rows of the products (S^T) took 131 us in the first case where the queries' as rows took 169, for up to 8 rows fill half of 16.
#include "gemm_api.h"
#include "paged.cuh"

#include <algorithm>
#include <string.h>

namespace mdb {

constexpr int PK = 128;                                       // keys of a tile: no more than a page has, or several pages
constexpr float PAGED_LOG2E = 1.4426950408889634f;

struct alignas(64) PagedMaps {
  CUtensorMap k, v;
};

// A warp has NT tiles of 8 rows; RG warps share the rows, and the others the keys of a tile
template <int DH, bool E4M3, int NT, int RG> struct PagedShape {
  // that multiply. Heads of 128 have room for the queries and sums of 8 rows in a warp; for 16 rows (168 registers, 90 to 110 bytes spilled) 8 sequences of 4000 with 32 rows took 49 us
  // (bf16 57) with four warps and two CTAs to an SM, with eight warps of 8 rows and one CTA 43 (45). Heads of 64 have room for 16: eight warps took 37 us instead of 33 there.
  static constexpr int WARPS = DH == 128 && RG > 1 ? 8 : 4;
  static constexpr int THREADS = (WARPS + 1) * 32;
  static constexpr int COLS = 64 / NT;                                // columns that the warps join at a time
  static constexpr int TILE = PK * DH * (E4M3 ? 1 : 2);               // K or V of a stage
  // per SM, with up to 192 KB of stages: 16 tokens over 16384, 64 / 8 heads of 64: three CTAs 76 us, two 94; 4 over 131072, heads of 128, where three would have two stages each: 150 and 143.
  // bf16 pages with heads of 128 and up to 8 rows have a stage of 64 KB to either CTA, so that copies run under the other CTA's work only, and 64 KB to spare: 16 over 16384 (32 / 8 heads)
  // 182 us, 5.9 TB/s, 32 over 0 to 16384 135 us, 5.4 TB/s.
  static constexpr int CTAS = WARPS == 8 ? 1 : NT == 1 && DH == 64 ? 3 : 2;
  static constexpr int STAGES = 192 * 1024 / CTAS / (2 * TILE);
  static_assert(STAGES >= 1);
  static constexpr int SLAB = WARPS * 8 * NT * COLS * 4;
  static constexpr int BYTES = STAGES * 2 * TILE + SLAB + 1024;
};

__device__ __forceinline__ float paged_max(float a, float b) {       // NaN stays
  float d;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(d) : "f"(a), "f"(b));
  return d;
}
__device__ __forceinline__ void paged_ldsm(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ void paged_ldsm_t(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
template <bool F16> __device__ __forceinline__ void paged_mma(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  if (F16)
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  else
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t paged_transpose(uint32_t x) {      // an 8 x 8 matrix of 16-bit elements over the warp
  uint32_t r;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(x));
  return r;
}
__device__ __forceinline__ uint32_t pack_f16x2(float lo, float hi) {
  const __half2 h = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&h);
}

// ---- the line of tiles: sequence after sequence, key head after key head, tile after tile ----
__device__ __forceinline__ int paged_length(const MdbPagedAttnArgs& a, int b) { return min(max(a.kv_len[b], 0), a.pages.most); }
__device__ __forceinline__ int paged_tiles(const MdbPagedAttnArgs& a) {      // of one key head; by a whole warp
  int total = 0;
  for (int b0 = 0; b0 < a.pages.B; b0 += 32) {
    const int b = b0 + (threadIdx.x & 31);
    total += __reduce_add_sync(0xffffffffu, b < a.pages.B ? static_cast<unsigned>(paged_length(a, b) + PK - 1) / PK : 0u);
  }
  return total;
}
// The line's shares: `ctas` of them, the first `more` with a tile more than the others. 32-bit divisions only, for they stand before the first load: with those of 64 bits the
// first tile was there 11300 cycles after a CTA's start, without them 10300 (cold caches), and 32 tokens over 0 to 16384 positions took 87 us instead of 80.
struct PagedShares {
  int ctas, each, more;
  __device__ __forceinline__ PagedShares(int line, int grid) : ctas(min(grid, line)), each(line / max(ctas, 1)), more(line - each * ctas) {}
  __device__ __forceinline__ int first(int cta) const { return cta * each + min(cta, more); }
  __device__ __forceinline__ int cta_of(int tile) const {
    const int early = more * (each + 1);
    return tile < early ? tile / (each + 1) : more + (tile - early) / each;
  }
};
struct PagedPlace {
  int b, g, t, length, tiles;
  // of tile `at` on the line; by a whole warp
  __device__ __forceinline__ void seek(const MdbPagedAttnArgs& a, int at) {
    const int lane = threadIdx.x & 31, target = at / a.pages.Hkv;
    int before = 0;
    b = 0;
    length = tiles = 0;
    for (int b0 = 0; b0 < a.pages.B; b0 += 32) {
      const int mine = b0 + lane < a.pages.B ? paged_length(a, b0 + lane) : 0, n = (mine + PK - 1) / PK;
      int upto = n;
#pragma unroll
      for (int m = 1; m < 32; m <<= 1) {
        const int other = __shfl_up_sync(0xffffffffu, upto, m);
        if (lane >= m) upto += other;
      }
      const uint32_t behind = __ballot_sync(0xffffffffu, before + upto > target);
      if (behind != 0) {
        const int from = __ffs(behind) - 1;
        b = b0 + from;
        length = __shfl_sync(0xffffffffu, mine, from);
        tiles = __shfl_sync(0xffffffffu, n, from);
        before += __shfl_sync(0xffffffffu, upto, from) - tiles;
        break;
      }
      before += __shfl_sync(0xffffffffu, upto, 31);
    }
    const int rest = at - before * a.pages.Hkv;
    g = tiles > 0 ? rest / tiles : 0;
    t = rest - g * tiles;
  }
  __device__ __forceinline__ void next_segment(const MdbPagedAttnArgs& a) {
    t = 0;
    if (++g < a.pages.Hkv) return;
    g = 0;
    do {
      if (++b >= a.pages.B) return;
      length = paged_length(a, b);
      tiles = (length + PK - 1) / PK;
    } while (tiles == 0);
  }
};

// parts: two per CTA, of the first and of the last segment of its tiles: [ctas][2][rows][DH] sums, then [ctas][2][rows][2] references and divisors
struct PagedParts {
  float* sums; float* tops;
};

template <int DH, bool E4M3, int NT, int RG>
__global__ void __launch_bounds__(PagedShape<DH, E4M3, NT, RG>::THREADS, PagedShape<DH, E4M3, NT, RG>::CTAS)
paged_step_kernel(const __grid_constant__ PagedMaps maps, const __grid_constant__ MdbPagedAttnArgs a, const PagedParts parts) {
  using Shape = PagedShape<DH, E4M3, NT, RG>;
  constexpr int TILE = Shape::TILE, STAGES = Shape::STAGES, BOX = PK * 128, WARPS = Shape::WARPS, COLS = Shape::COLS;
  constexpr int WR = 8 * NT, ROWS = WR * RG, PER_TILE = WARPS / RG, WK = PK / PER_TILE;      // rows of a warp, of all; warps that share the keys, and keys of a warp
  constexpr int DM = DH / 16;                                                                   // tiles of 16 columns
  constexpr float ABOVE = E4M3 ? 7.f : 0.f;                                                     // the reference stays so far below the first maximum

  extern __shared__ uint8_t smem_raw[];
  __shared__ uint64_t full[STAGES], empty[STAGES];
  __shared__ uchar2 scales[STAGES][PK / 16];
  __shared__ int abort_s;
  __shared__ float part_m[WARPS][WR], part_l[WARPS][WR];
  uint8_t* smem = smem_raw + (((smem_u32(smem_raw) + 1023u) & ~1023u) - smem_u32(smem_raw));
  float* slab = reinterpret_cast<float*>(smem + STAGES * 2 * TILE);

  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const MdbPages& pg = a.pages;
  if (warp == WARPS && lane == 0) {
    tma_prefetch_desc(&maps.k);
    tma_prefetch_desc(&maps.v);
  }
  if (threadIdx.x == 0) {
    for (int s = 0; s < STAGES; ++s) {
      mbar_init(&full[s], E4M3 ? 2 : 1);      // the copies, and the scales
      mbar_init(&empty[s], WARPS);
    }
    abort_s = 0;
    fence_mbar_init();
  }
  PagedPlace at;
  int n;
  if (parts.sums == nullptr) {      // one sequence and head
    at.b = blockIdx.x / pg.Hkv;
    at.g = blockIdx.x - at.b * pg.Hkv;
    at.t = 0;
    at.length = paged_length(a, at.b);
    n = at.tiles = (at.length + PK - 1) / PK;
    __syncthreads();
    if (n == 0) {
      const int rep = a.H / pg.Hkv;
      for (int e = threadIdx.x; e < rep * a.Sq * (DH / 8); e += Shape::THREADS) {
        const int r = e / (DH / 8);
        *reinterpret_cast<uint4*>(static_cast<__nv_bfloat16*>(a.o) + at.b * a.o_strides[0] + (r / rep) * a.o_strides[1] + (at.g * rep + r % rep) * a.o_strides[2] + e % (DH / 8) * 8) = make_uint4(0, 0, 0, 0);
      }
      return;
    }
  } else {
    const PagedShares shares(paged_tiles(a) * pg.Hkv, gridDim.x);
    const int cta = blockIdx.x, line_first = cta < shares.ctas ? shares.first(cta) : 0;
    at.seek(a, line_first);
    __syncthreads();
    if (cta >= shares.ctas) return;
    n = shares.first(cta + 1) - line_first;
  }

  if (warp == WARPS) {
    const int per_tile = PK >> pg.shift, rows = pg.P;            // boxes of a tile, keys of a box
    const uint32_t box_bytes = rows * DH * (E4M3 ? 1 : 2);
    int window = 0, page = -1;                                              // this lane's place of the table: window + lane
    uint32_t sc = 0;
    bool ok = true, fresh = true;
    int i = 0;
    for (; i < n; ++i) {
      const int first_index = at.t * PK >> pg.shift;
      if (fresh || first_index + per_tile > window + 32) {
        window = first_index;
        const int index = window + lane;
        const bool needed = index <= (at.length - 1) >> pg.shift;
        page = needed ? page_of(pg, at.b, index) : -1;
        if (needed && page < 0) report_status(pg.status, STATUS_BOUNDS, 182, at.b);
        if (E4M3) {
          sc = 0;
          if (page >= 0) sc = pg.k_scale[page * pg.scale_strides[0] + at.g] | pg.v_scale[page * pg.scale_strides[1] + at.g] << 8;
        }
        fresh = false;
      }
      const int st = i % STAGES;
      ok = __all_sync(0xffffffffu, mbar_wait(&empty[st], ((i / STAGES) & 1) ^ 1u, &abort_s));
      if (!ok) {
        if (lane == 0) report_status(pg.status, STATUS_TIMEOUT, 183, i);
        break;
      }
      const int keys = min(at.length - at.t * PK, PK), boxes = (keys + rows - 1) >> pg.shift;
      const int mine = __shfl_sync(0xffffffffu, page, (first_index - window + min(lane, per_tile - 1)) & 31);
      __syncwarp();
      if (lane == 0) mbar_expect_tx(&full[st], 2 * boxes * box_bytes);
      __syncwarp();
      if (lane < boxes) {
        uint8_t* to = smem + st * 2 * TILE;
        if (E4M3) {
          tma_load_4d(to + lane * box_bytes, &maps.k, &full[st], 0, 0, at.g, mine);
          tma_load_4d(to + TILE + lane * box_bytes, &maps.v, &full[st], 0, 0, at.g, mine);
        } else {
#pragma unroll
          for (int d = 0; d < DH / 64; ++d) {
            tma_load_4d(to + d * BOX + lane * rows * 128, &maps.k, &full[st], d * 64, 0, at.g, mine);
            tma_load_4d(to + TILE + d * BOX + lane * rows * 128, &maps.v, &full[st], d * 64, 0, at.g, mine);
          }
        }
      }
      if (E4M3) {      // behind the copies, which need not wait for them
        const uint32_t s = __shfl_sync(0xffffffffu, sc, ((at.t * PK + (lane & 7) * 16 >> pg.shift) - window) & 31);
        if (lane < PK / 16) scales[st][lane] = make_uchar2(s & 255, s >> 8);
        __syncwarp();
        if (lane == 0) mbar_arrive(&full[st]);
      }
      __syncwarp();
      if (++at.t == at.tiles) {
        at.next_segment(a);
        fresh = true;
      }
    }
    if (!ok && lane == 0) {      // the copies on the way land before the memory is given up
      for (int j = max(0, i - STAGES); j < i; ++j) {
        const uint64_t t0 = globaltimer_ns();
        while (!mbar_try_wait(&full[j % STAGES], (j / STAGES) & 1) && globaltimer_ns() - t0 < 5000000ull) {
        }
      }
    }
    __syncwarp();
    return;
  }

  const int rg = warp / PER_TILE, part = warp % PER_TILE;
  const int tq = lane & 3, gq = lane >> 2;
  const int rep = a.H / pg.Hkv, rows = rep * a.Sq;
  // Key j of a group of eight lies in this row of the stage: with a row of 128 bytes, lanes that read 16 bytes each at once then hit all banks (see the swizzle).
  const auto key_of = [](int j) { return E4M3 && DH == 128 ? (j >> 1) + 4 * (j & 1) : j; };
  bool ok = true;
  for (int i = 0, segment = 0; i < n; ++segment) {
    const int b = at.b, g = at.g, first_tile = at.t, end = at.length, start = end - a.Sq;
    const int count = min(at.tiles - first_tile, n - i);
    uint32_t q[NT][DH / 16][2];
    float sl2[NT][2];                                                   // of the rows 2 t, 2 t + 1 of a tile of 8, whose scores this lane has
    int p_row[NT][2];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      const int r = rg * WR + nt * 8 + gq;
      const __nv_bfloat16* p = static_cast<const __nv_bfloat16*>(a.q) + b * a.q_strides[0] + (r / rep) * a.q_strides[1] + (g * rep + r % rep) * a.q_strides[2];
      float mine = a.scale * PAGED_LOG2E;
      if (E4M3) {
        // k-step 4 c + s: columns 16 (4 c + t) + 4 s .. + 3 belong to lane t
        float most = 0.f;
#pragma unroll
        for (int c = 0; c < DH / 64; ++c)
#pragma unroll
          for (int x = 0; x < 4; x += 2) {
            const uint4 u = r < rows ? *reinterpret_cast<const uint4*>(p + 16 * (4 * c + tq) + 4 * x) : make_uint4(0, 0, 0, 0);
            q[nt][4 * c + x][0] = u.x;
            q[nt][4 * c + x][1] = u.y;
            q[nt][4 * c + x + 1][0] = u.z;
            q[nt][4 * c + x + 1][1] = u.w;
          }
#pragma unroll
        for (int kk = 0; kk < DH / 16; ++kk)
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const float2 f = unpack_bf16x2(q[nt][kk][e]);
            most = fmaxf(most, fmaxf(fabsf(f.x), fabsf(f.y)));      // NaN and infinity come through by themselves
          }
        most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, 1));
        most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, 2));
        const int e = min(max(static_cast<int>(__float_as_uint(most) >> 23), 1), 253);
        const float f = scale_inverse(e);
        mine *= scale_value(e);
#pragma unroll
        for (int kk = 0; kk < DH / 16; ++kk)
#pragma unroll
          for (int y = 0; y < 2; ++y) {
            const float2 x = unpack_bf16x2(q[nt][kk][y]);
            q[nt][kk][y] = pack_f16x2(x.x * f, x.y * f);
          }
      } else {
#pragma unroll
        for (int kk = 0; kk < DH / 16; ++kk) {
          q[nt][kk][0] = r < rows ? *reinterpret_cast<const uint32_t*>(p + kk * 16 + 2 * tq) : 0u;
          q[nt][kk][1] = r < rows ? *reinterpret_cast<const uint32_t*>(p + kk * 16 + 2 * tq + 8) : 0u;
        }
      }
#pragma unroll
      for (int y = 0; y < 2; ++y) {
        sl2[nt][y] = __shfl_sync(0xffffffffu, mine, 4 * (2 * tq + y));
        p_row[nt][y] = start + (rg * WR + nt * 8 + 2 * tq + y) / rep;
      }
    }
    float o[DM][NT][4];
#pragma unroll
    for (int d = 0; d < DM; ++d)
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int e = 0; e < 4; ++e) o[d][nt][e] = 0.f;
    float m[NT][2], l[NT][2];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      m[nt][0] = m[nt][1] = -INFINITY;
      l[nt][0] = l[nt][1] = 0.f;
    }
    float u[NT][2];                                                    // o is in units of 2^(u - 127), a whole number for each row
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) u[nt][0] = u[nt][1] = 145.f;      // 2^(ev - u) is a number for any ev

    for (int tile = first_tile; tile < first_tile + count; ++tile, ++i) {
      const int st = i % STAGES;
      if (ok) ok = __all_sync(0xffffffffu, mbar_wait(&full[st], (i / STAGES) & 1, &abort_s));
      if (!ok) continue;
      const uint8_t* sk = smem + st * 2 * TILE;
      uint8_t* sv = smem + st * 2 * TILE + TILE;
#pragma unroll 1
      for (int k32 = part * WK; k32 < part * WK + WK && rg * WR < rows; k32 += 32) {      // row in the stage; a warp without rows only gives the stages back
        const int kb = tile * PK + k32;                                 // key
        if (kb >= end) break;
        if (kb + 32 > end) {
          const int r = k32 + lane;
          if (kb + lane >= end) {
            if (E4M3) {
              const int line_ = r * DH / 128, chunk = (r * DH % 128) / 16;
#pragma unroll
              for (int c = 0; c < DH / 16; ++c) *reinterpret_cast<uint4*>(sv + line_ * 128 + (((chunk + c) ^ (line_ & 7)) << 4)) = make_uint4(0, 0, 0, 0);
            } else {
              for (int x = 0; x < DH / 64; ++x)
                for (int c = 0; c < 8; ++c) *reinterpret_cast<uint4*>(sv + x * BOX + r * 128 + c * 16) = make_uint4(0, 0, 0, 0);
            }
          }
          __syncwarp();
          fence_proxy_async_smem();
        }
        // S^T of 2 x 16 keys: this lane has keys gq and gq + 8, rows 2 t and 2 t + 1
        float x[2][NT][4];
#pragma unroll
        for (int s = 0; s < 2; ++s) {
#pragma unroll
          for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int e = 0; e < 4; ++e) x[s][nt][e] = 0.f;
          if (E4M3) {
#pragma unroll
            for (int c = 0; c < DH / 64; ++c) {
              uint32_t w[2][4];
#pragma unroll
              for (int y = 0; y < 2; ++y) {
                const int r = k32 + s * 16 + y * 8 + key_of(gq), line_ = r * DH / 128, chunk = (r * DH % 128) / 16 + 4 * c + tq;
                *reinterpret_cast<uint4*>(w[y]) = *reinterpret_cast<const uint4*>(sk + line_ * 128 + ((chunk ^ (line_ & 7)) << 4));
              }
#pragma unroll
              for (int z = 0; z < 4; ++z) {
                const uint32_t k4[4] = {e4m3x2_to_f16x2(static_cast<uint16_t>(w[0][z])), e4m3x2_to_f16x2(static_cast<uint16_t>(w[1][z])),
                                        e4m3x2_to_f16x2(static_cast<uint16_t>(w[0][z] >> 16)), e4m3x2_to_f16x2(static_cast<uint16_t>(w[1][z] >> 16))};
#pragma unroll
                for (int nt = 0; nt < NT; ++nt) paged_mma<true>(x[s][nt], k4, q[nt][4 * c + z][0], q[nt][4 * c + z][1]);
              }
            }
          } else {
            const int r = k32 + s * 16 + (lane & 15);
#pragma unroll
            for (int kk = 0; kk < DH / 16; ++kk) {
              uint32_t w[4];
              const int c = (kk & 3) * 2 + (lane >> 4);
              paged_ldsm(w, smem_u32(sk) + (kk >> 2) * BOX + r * 128 + ((c ^ (r & 7)) << 4));
#pragma unroll
              for (int nt = 0; nt < NT; ++nt) paged_mma<false>(x[s][nt], w, q[nt][kk][0], q[nt][kk][1]);
            }
          }
        }
        float ks[2] = {1.f, 1.f}, ev[2] = {0.f, 0.f};                  // unit of the keys, byte of the values' (a page behind the end: 0)
        bool apart = false;
        if (E4M3) {
          const uchar2 sc[2] = {scales[st][k32 / 16], scales[st][k32 / 16 + 1]};
          apart = sc[0].y != sc[1].y;      // the same in the whole warp
#pragma unroll
          for (int s = 0; s < 2; ++s) {
            ks[s] = scale_value(sc[s].x);
            ev[s] = sc[s].y;
          }
        }
        const bool whole = kb + 31 <= start && kb + 32 <= end;
        bool raise = false;
        float top[NT][2], big[NT][2];     // the largest of the scores, and of the scores plus ev
        float2 mul[2][NT];                // of the rows 2 t, 2 t + 1; not 0, for -inf * 0 is not -inf
        const float most_ev = fmaxf(ev[0], ev[1]);
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
          top[nt][0] = top[nt][1] = big[nt][0] = big[nt][1] = -INFINITY;
#pragma unroll
          for (int s = 0; s < 2; ++s) {
            mul[s][nt] = make_float2(fmaxf(sl2[nt][0] * ks[s], 0x1p-126f), fmaxf(sl2[nt][1] * ks[s], 0x1p-126f));
            if (!whole) {
#pragma unroll
              for (int e = 0; e < 4; ++e) {
                const int j = kb + s * 16 + key_of(gq) + 8 * (e >> 1);
                if (!(j <= p_row[nt][e & 1] && j < end)) x[s][nt][e] = -INFINITY;
              }
            }
            const float t[2] = {paged_max(x[s][nt][0], x[s][nt][2]) * mul[s][nt].x, paged_max(x[s][nt][1], x[s][nt][3]) * mul[s][nt].y};
#pragma unroll
            for (int y = 0; y < 2; ++y) {
              top[nt][y] = paged_max(top[nt][y], t[y]);
              if (E4M3) big[nt][y] = paged_max(big[nt][y], t[y] + ev[s]);
            }
          }
#pragma unroll
          for (int y = 0; y < 2; ++y) {
#pragma unroll
            for (int z = 4; z < 32; z <<= 1) top[nt][y] = paged_max(top[nt][y], __shfl_xor_sync(0xffffffffu, top[nt][y], z));
            top[nt][y] -= ABOVE;
            // The reference is raised when outgrown by more than 2^8, and with the first key that the row sees; NaN is kept. u is set when the weights have outgrown it, and
            // where m is; it stays within 2^118 of every unit, so that 2^(ev - u) is a number.
            raise = raise || !(top[nt][y] <= m[nt][y] + 8.f);
          }
        }
        if (E4M3) {
          if (apart) {
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
              for (int y = 0; y < 2; ++y) {
#pragma unroll
                for (int z = 4; z < 32; z <<= 1) big[nt][y] = paged_max(big[nt][y], __shfl_xor_sync(0xffffffffu, big[nt][y], z));
                big[nt][y] -= ABOVE;
              }
          } else {
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
              for (int y = 0; y < 2; ++y) big[nt][y] = top[nt][y] + ev[0];
          }
#pragma unroll
          for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int y = 0; y < 2; ++y) raise = raise || !(big[nt][y] <= m[nt][y] + (u[nt][y] + 8.f)) || most_ev > u[nt][y] + 118.f;
        }
        if (__any_sync(0xffffffffu, raise)) {
          float fo[NT][2];
#pragma unroll
          for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int y = 0; y < 2; ++y) {
              float down = 0.f;             // log2 of what m changes everything by
              if (!(top[nt][y] <= m[nt][y] + 8.f)) {
                down = m[nt][y];
                m[nt][y] = paged_max(m[nt][y], top[nt][y]);
                down -= m[nt][y];
              }
              fo[nt][y] = exp2f(down);
              l[nt][y] *= fo[nt][y];
              if (E4M3) {                   // a number in any case: a row without keys so far keeps its u, one of NaN has no use for it
                const float now = ceilf(fmaxf(fmaxf(u[nt][y] + down, big[nt][y] - m[nt][y]), most_ev - 110.f));
                fo[nt][y] = exp2f(down + (u[nt][y] - now));
                u[nt][y] = now;
              }
            }
#pragma unroll
          for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int d = 0; d < DM; ++d)
#pragma unroll
              for (int e = 0; e < 4; ++e) o[d][nt][e] *= fo[nt][e & 1];
        }
        // P^T as the B operand: keys 2 t, 2 t + 1 (and 8 more) of row gq, which is the transpose of what the lane has
        uint32_t ph[2][NT][2], pl[2][NT][2];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
          const float2 less = make_float2(m[nt][0] == -INFINITY ? 0.f : -m[nt][0], m[nt][1] == -INFINITY ? 0.f : -m[nt][1]);
          float2 sum = make_float2(l[nt][0], l[nt][1]);
#pragma unroll
          for (int s = 0; s < 2; ++s) {
            const float2 into = E4M3 ? make_float2(ex2_approx(ev[s] - u[nt][0]), ex2_approx(ev[s] - u[nt][1])) : make_float2(1.f, 1.f);
#pragma unroll
            for (int y = 0; y < 2; ++y) {
              const float2 t = ffma2(make_float2(x[s][nt][2 * y], x[s][nt][2 * y + 1]), mul[s][nt], less);
              const float2 p = make_float2(ex2_approx(t.x), ex2_approx(t.y));
              sum = fadd2(sum, p);
              if (E4M3) {
                const float2 q2 = fmul2(p, into);
                ph[s][nt][y] = paged_transpose(pack_f16x2(q2.x, q2.y));
              } else {
                const uint32_t h = pack_bf16x2(p.x, p.y);
                const float2 low = ffma2(unpack_bf16x2(h), make_float2(-1.f, -1.f), p);
                ph[s][nt][y] = paged_transpose(h);
                pl[s][nt][y] = paged_transpose(pack_bf16x2(low.x, low.y));
              }
            }
          }
          l[nt][0] = sum.x;
          l[nt][1] = sum.y;
        }
#pragma unroll
        for (int s = 0; s < 2; ++s) {
          const int kr = k32 + s * 16;
          if (E4M3) {
            // a tile's rows gq and gq + 8 are the columns 16 c + 2 gq and 16 c + 2 gq + 1
            const int r = kr + (lane & 8) + key_of(lane & 7), line_ = r * DH / 128;
#pragma unroll
            for (int c = 0; c < DM; c += 2) {
              uint32_t w[4];
              const int chunk = (r * DH % 128) / 16 + c + (lane >> 4);
              paged_ldsm_t(w, smem_u32(sv) + line_ * 128 + ((chunk ^ (line_ & 7)) << 4));
#pragma unroll
              for (int y = 0; y < 2; ++y) {
                const uint32_t b0 = __byte_perm(w[2 * y], 0, 0x3120), b1 = __byte_perm(w[2 * y + 1], 0, 0x3120);
                const uint32_t v4[4] = {e4m3x2_to_f16x2(static_cast<uint16_t>(b0)), e4m3x2_to_f16x2(static_cast<uint16_t>(b0 >> 16)),
                                        e4m3x2_to_f16x2(static_cast<uint16_t>(b1)), e4m3x2_to_f16x2(static_cast<uint16_t>(b1 >> 16))};
#pragma unroll
                for (int nt = 0; nt < NT; ++nt) paged_mma<true>(o[c + y][nt], v4, ph[s][nt][0], ph[s][nt][1]);
              }
            }
          } else {
            const int r = kr + (lane & 7) + 8 * (lane >> 4);
#pragma unroll
            for (int c = 0; c < DM; ++c) {
              uint32_t w[4];
              const int chunk = (c & 3) * 2 + (lane >> 3 & 1);
              paged_ldsm_t(w, smem_u32(sv) + (c >> 2) * BOX + r * 128 + ((chunk ^ (r & 7)) << 4));
#pragma unroll
              for (int nt = 0; nt < NT; ++nt) {
                paged_mma<false>(o[c][nt], w, ph[s][nt][0], ph[s][nt][1]);
                paged_mma<false>(o[c][nt], w, pl[s][nt][0], pl[s][nt][1]);
              }
            }
          }
        }
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(&empty[st]);
    }

    // the warps' parts meet in shared memory, COLS columns at a time
    // 8 bits: divisors are brought to [1, 2), and sums with them, so that these are no larger than the values
    float less[NT][2], units[NT][2];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int y = 0; y < 2; ++y) {
#pragma unroll
        for (int z = 4; z < 32; z <<= 1) l[nt][y] += __shfl_xor_sync(0xffffffffu, l[nt][y], z);
        if (E4M3) {
          const int e = min(max(static_cast<int>(__float_as_uint(l[nt][y]) >> 23), 1), 253);      // 0 (no key) and NaN stay as they are
          less[nt][y] = scale_inverse(e);
          units[nt][y] = exp2f(u[nt][y] - 127.f);
          l[nt][y] *= less[nt][y];
          m[nt][y] += e - 127;
        }
        if (gq == 0) {
          part_m[warp][nt * 8 + 2 * tq + y] = m[nt][y];
          part_l[warp][nt * 8 + 2 * tq + y] = l[nt][y];
        }
      }
    const bool complete = first_tile == 0 && count == at.tiles;
    const long long slot = 2ll * blockIdx.x + (segment > 0 ? 1 : 0);
#pragma unroll
    for (int c0 = 0; c0 < DH; c0 += COLS) {
#pragma unroll
      for (int y = 0; y < COLS / 16; ++y)
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
          const float (&v)[4] = o[c0 / 16 + y][nt];
          float* mine = slab + (warp * WR + nt * 8 + 2 * tq) * COLS + 16 * y;
          if (E4M3) {
            *reinterpret_cast<float2*>(mine + 2 * gq) = make_float2(v[0] * less[nt][0] * units[nt][0], v[2] * less[nt][0] * units[nt][0]);
            *reinterpret_cast<float2*>(mine + COLS + 2 * gq) = make_float2(v[1] * less[nt][1] * units[nt][1], v[3] * less[nt][1] * units[nt][1]);
          } else {
            mine[gq] = v[0];
            mine[gq + 8] = v[2];
            mine[COLS + gq] = v[1];
            mine[COLS + gq + 8] = v[3];
          }
        }
      asm volatile("bar.sync 1, %0;" ::"n"(WARPS * 32) : "memory");
      for (int e = threadIdx.x; e < rows * (COLS / 4); e += WARPS * 32) {
        const int r = e / (COLS / 4), w0 = (r / WR) * PER_TILE, rr = r % WR, c = e % (COLS / 4) * 4;
        float top = part_m[w0][rr];
#pragma unroll
        for (int w = 1; w < PER_TILE; ++w) top = paged_max(top, part_m[w0 + w][rr]);
        float4 s = make_float4(0.f, 0.f, 0.f, 0.f);
        float sum = 0.f;
#pragma unroll
        for (int w = 0; w < PER_TILE; ++w) {
          const float f = part_m[w0 + w][rr] == -INFINITY ? 0.f : exp2f(part_m[w0 + w][rr] - top);
          const float4 v = *reinterpret_cast<const float4*>(slab + ((w0 + w) * WR + rr) * COLS + c);
          s.x += f * v.x;
          s.y += f * v.y;
          s.z += f * v.z;
          s.w += f * v.w;
          sum += f * part_l[w0 + w][rr];
        }
        if (!ok) continue;
        if (complete) {
          const float inv = top == -INFINITY ? 0.f : 1.f / sum;
          uint2 w;
          w.x = pack_bf16x2(s.x * inv, s.y * inv);
          w.y = pack_bf16x2(s.z * inv, s.w * inv);
          if (top == -INFINITY) w = make_uint2(0, 0);
          *reinterpret_cast<uint2*>(static_cast<__nv_bfloat16*>(a.o) + b * a.o_strides[0] + (r / rep) * a.o_strides[1] + (g * rep + r % rep) * a.o_strides[2] + c0 + c) = w;
        } else {
          *reinterpret_cast<float4*>(parts.sums + (slot * ROWS + r) * DH + c0 + c) = s;
          if (c0 == 0 && c == 0) *reinterpret_cast<float2*>(parts.tops + (slot * ROWS + r) * 2) = make_float2(top, sum);
        }
      }
      asm volatile("bar.sync 1, %0;" ::"n"(WARPS * 32) : "memory");
    }
    at.t = first_tile + count;
    if (at.t == at.tiles) at.next_segment(a);
  }
  if (!ok && lane == 0) report_status(pg.status, STATUS_TIMEOUT, 184, n);
}

// A row to a warp, or to all four of a block where a row has many parts: the parts of its key head, in order. What they need to know they find out while the first kernel
// runs. Rows of sequences without keys are zero.
constexpr int PJ_THREADS = 128;
template <int DH, int WARPS>
__global__ void __launch_bounds__(PJ_THREADS)
paged_join_kernel(const __grid_constant__ MdbPagedAttnArgs a, const PagedParts parts, const int grid, const int part_rows) {
  constexpr int LANES = DH / 4, IN_WARP = 32 / LANES, GROUPS = WARPS * IN_WARP;
  __shared__ float tops[4], sums[4];
  __shared__ float4 slab[4][LANES];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, c = lane % LANES, group = warp % WARPS * IN_WARP + lane / LANES;
  const long long row = blockIdx.x * (4ll / WARPS) + warp / WARPS;
  const int per = a.Sq * a.H;
  const bool in = row < static_cast<long long>(a.pages.B) * per;
  const int b = in ? static_cast<int>(row / per) : 0, rest = in ? static_cast<int>(row - static_cast<long long>(b) * per) : 0, h = rest % a.H, i = rest / a.H;
  const int rep = a.H / a.pages.Hkv, g = h / rep, r = i * rep + h % rep;
  int before = 0, total = 0;                          // tiles of a key head before this sequence, in all
  for (int b0 = 0; b0 < a.pages.B; b0 += 32) {
    const unsigned n = b0 + lane < a.pages.B ? static_cast<unsigned>(paged_length(a, b0 + lane) + PK - 1) / PK : 0u;
    total += __reduce_add_sync(0xffffffffu, n);
    before += __reduce_add_sync(0xffffffffu, b0 + lane < b ? n : 0u);
  }
  const int tiles = (paged_length(a, b) + PK - 1) / PK, u0 = before * a.pages.Hkv + g * tiles;
  const PagedShares shares(max(total * a.pages.Hkv, 1), grid);
  const int first = shares.cta_of(u0), last = shares.cta_of(u0 + max(tiles, 1) - 1);
  const bool first_of_all = shares.first(first) == u0;
  __nv_bfloat16* out = static_cast<__nv_bfloat16*>(a.o) + b * a.o_strides[0] + i * a.o_strides[1] + h * a.o_strides[2];
  asm volatile("griddepcontrol.wait;" ::: "memory");      // by all: this kernel must not end before the one whose parts it joins
  if (in && tiles == 0 && group == 0) *reinterpret_cast<uint2*>(out + c * 4) = make_uint2(0, 0);
  const bool joined = in && tiles > 0 && first < last;
  if (!joined) return;                                     // the same in a warp, and with four warps to a row in the block
  float top = -INFINITY, sum = 0.f;
  float4 s = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 4
  for (int k = first + group; k <= last; k += GROUPS) {
    const long long slot = 2ll * k + (k == first && !first_of_all ? 1 : 0);
    const float2 ml = *reinterpret_cast<const float2*>(parts.tops + (slot * part_rows + r) * 2);
    const float4 v = *reinterpret_cast<const float4*>(parts.sums + (slot * part_rows + r) * DH + c * 4);
    if (ml.x == -INFINITY) continue;
    const float up = paged_max(top, ml.x), f = top == -INFINITY ? 0.f : exp2f(top - up), w = exp2f(ml.x - up);
    s.x = s.x * f + v.x * w;
    s.y = s.y * f + v.y * w;
    s.z = s.z * f + v.z * w;
    s.w = s.w * f + v.w * w;
    sum = sum * f + ml.y * w;
    top = up;
  }
  const auto join = [&](float top2, float sum2, float4 v) {
    const float up = paged_max(top, top2), f = top == -INFINITY ? 0.f : exp2f(top - up), w = top2 == -INFINITY ? 0.f : exp2f(top2 - up);
    s.x = s.x * f + v.x * w;
    s.y = s.y * f + v.y * w;
    s.z = s.z * f + v.z * w;
    s.w = s.w * f + v.w * w;
    sum = sum * f + sum2 * w;
    top = up;
  };
  if (IN_WARP == 2) {
    const float4 v = make_float4(__shfl_down_sync(0xffffffffu, s.x, 16), __shfl_down_sync(0xffffffffu, s.y, 16), __shfl_down_sync(0xffffffffu, s.z, 16), __shfl_down_sync(0xffffffffu, s.w, 16));
    const float top2 = __shfl_down_sync(0xffffffffu, top, 16), sum2 = __shfl_down_sync(0xffffffffu, sum, 16);
    if (lane < 16) join(top2, sum2, v);
  }
  if (WARPS > 1) {
    if (lane < LANES) slab[warp][lane] = s;
    if (lane == 0) {
      tops[warp] = top;
      sums[warp] = sum;
    }
    __syncthreads();
    if (warp > 0) return;
#pragma unroll
    for (int w = 1; w < WARPS; ++w) join(tops[w], sums[w], slab[w][c]);
  }
  if (lane >= LANES) return;
  uint2 w = make_uint2(0, 0);
  if (top != -INFINITY) {
    const float inv = 1.f / sum;
    w = make_uint2(pack_bf16x2(s.x * inv, s.y * inv), pack_bf16x2(s.z * inv, s.w * inv));
  }
  *reinterpret_cast<uint2*>(out + c * 4) = w;
}

static int pages_map(CUtensorMap* m, const void* pool, const MdbPages& p, const long long* strides, bool e4m3) {
  if (e4m3) {      // lines of 128 bytes: a key of 128, two of 64
    const int lines = p.P * p.Dh / 128;
    int64_t ext[4] = {128, lines, p.Hkv, p.count};
    int64_t str[4] = {1, 128, strides[1], strides[0]};
    int box[4] = {128, std::min(p.P, PK) * p.Dh / 128, 1, 1};
    return mdb_make_tmap(m, pool, 1, 4, ext, str, box, 1);
  }
  int64_t ext[4] = {p.Dh, p.P, p.Hkv, p.count};
  int64_t str[4] = {2, p.Dh * 2, strides[1] * 2, strides[0] * 2};
  int box[4] = {64, std::min(p.P, PK), 1, 1};
  return mdb_make_tmap(m, pool, 2, 4, ext, str, box, 1);
}

// rows that the kernel has room for: 8, 16, 32 or 64
static int step_rows(const MdbPagedAttnArgs& a) {
  const int rows = a.Sq * (a.H / a.pages.Hkv);
  return rows <= 8 ? 8 : rows <= 16 ? 16 : rows <= 32 ? 32 : 64;
}
// One CTA for each sequence and key head, and nothing to join: the longest has four tiles at most. In us, so / shared out and joined: one token over 300 positions of 8 heads of
// 128 10.2 / 12.3, 8 over 500 12.3 / 16.4, 64 over 500 28.7 / 30.7, 16 over 300 of 8 heads of 64 10.2 / 14.4; with four tiles, 512 positions, 12.3 / 12.3.
static bool is_whole(const MdbPagedAttnArgs& a) { return a.pages.most <= 4 * PK; }
// As many CTAs as the SMs hold (see PagedShape), or one per tile where there are fewer
static int step_ctas(const MdbPagedAttnArgs& a) {
  const long long tiles = static_cast<long long>(a.pages.B) * a.pages.Hkv * ((a.pages.most + PK - 1) / PK);
  return static_cast<int>(std::max(1ll, std::min(tiles, (a.pages.Dh == 64 ? (step_rows(a) == 8 ? 3ll : 2ll) : step_rows(a) == 8 ? 2ll : 1ll) * device_sm_count())));
}

template <int DH, bool E4M3, int NT, int RG>
static int launch_step(const PagedMaps& maps, const MdbPagedAttnArgs& a, cudaStream_t st) {
  auto kern = paged_step_kernel<DH, E4M3, NT, RG>;
  static bool ready[64];
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e == cudaSuccess && (dev >= 64 || !ready[dev])) {
    e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, PagedShape<DH, E4M3, NT, RG>::BYTES);
    if (e == cudaSuccess && dev < 64) ready[dev] = true;
  }
  if (e != cudaSuccess) return static_cast<int>(e);
  if (is_whole(a)) {
    kern<<<a.pages.B * a.pages.Hkv, PagedShape<DH, E4M3, NT, RG>::THREADS, PagedShape<DH, E4M3, NT, RG>::BYTES, st>>>(maps, a, PagedParts{nullptr, nullptr});
    return static_cast<int>(cudaGetLastError());
  }
  const int ctas = step_ctas(a);
  constexpr int ROWS = 8 * NT * RG;
  const PagedParts parts = {a.ws, a.ws + 2ll * ctas * ROWS * DH};
  kern<<<ctas, PagedShape<DH, E4M3, NT, RG>::THREADS, PagedShape<DH, E4M3, NT, RG>::BYTES, st>>>(maps, a, parts);
  if ((e = cudaGetLastError()) != cudaSuccess) return static_cast<int>(e);
  cudaLaunchConfig_t c;
  memset(&c, 0, sizeof(c));
  // Four warps to a row where it has more than eight parts on average, as one long sequence has: there a warp alone would have ten loads behind one another.
  const bool many = ctas > 8ll * a.pages.B * a.pages.Hkv;
  const long long all = static_cast<long long>(a.pages.B) * a.Sq * a.H;
  c.gridDim = dim3(static_cast<unsigned>(many ? all : (all + 3) / 4));
  c.blockDim = dim3(PJ_THREADS);
  c.stream = st;
  cudaLaunchAttribute at;
  at.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at.val.programmaticStreamSerializationAllowed = 1;
  c.attrs = &at;
  c.numAttrs = 1;
  return static_cast<int>(cudaLaunchKernelEx(&c, many ? paged_join_kernel<DH, 4> : paged_join_kernel<DH, 1>, a, parts, ctas, ROWS));
}
template <int DH, bool E4M3>
static int launch_paged(const MdbPagedAttnArgs& a, cudaStream_t st) {
  PagedMaps maps;
  int r = pages_map(&maps.k, a.pages.k, a.pages, a.pages.k_strides, E4M3);
  if (r) return 2000 + r;
  r = pages_map(&maps.v, a.pages.v, a.pages, a.pages.v_strides, E4M3);
  if (r) return 3000 + r;
  const int rows = step_rows(a);
  constexpr int NT = DH == 64 ? 2 : 1;
  if (rows == 8) return launch_step<DH, E4M3, 1, 1>(maps, a, st);
  if (rows == 16) return launch_step<DH, E4M3, NT, 2 / NT>(maps, a, st);
  return rows == 32 ? launch_step<DH, E4M3, NT, 4 / NT>(maps, a, st) : launch_step<DH, E4M3, NT, 8 / NT>(maps, a, st);
}

// ---- parts of prompts: the pages in one piece, for the kernels of whole prompts ----
template <int DH, bool E4M3>
__global__ void __launch_bounds__(256)
paged_gather_kernel(const __grid_constant__ MdbPagedAttnArgs a, __nv_bfloat16* __restrict__ k, __nv_bfloat16* __restrict__ v, int* __restrict__ lengths) {
  const MdbPages& pg = a.pages;
  constexpr int LANES = DH / 16;
  const int b = blockIdx.y, length = paged_length(a, b), per_key = pg.Hkv * LANES;
  if (blockIdx.x == 0 && threadIdx.x == 0) {
    lengths[b] = length;
    lengths[pg.B + b] = length - a.Sq;
  }
  for (long long e = blockIdx.x * 256ll + threadIdx.x; e < static_cast<long long>(length) * per_key; e += gridDim.x * 256ll) {
    const int j = static_cast<int>(e / per_key), rest = static_cast<int>(e - static_cast<long long>(j) * per_key), g = rest / LANES, c = rest % LANES * 16;
    const int page = page_of(pg, b, j >> pg.shift);
    if (page < 0) report_status(pg.status, STATUS_BOUNDS, 185, b);
#pragma unroll
    for (int kv = 0; kv < 2; ++kv) {
      uint4 u[2] = {make_uint4(0, 0, 0, 0), make_uint4(0, 0, 0, 0)};
      if (page >= 0) {
        const long long* s = kv ? pg.v_strides : pg.k_strides;
        const long long from = page * s[0] + g * s[1] + (j & (pg.P - 1)) * DH + c;
        if (E4M3) {
          const float f = scale_value((kv ? pg.v_scale : pg.k_scale)[page * pg.scale_strides[kv] + g]);
          const uint4 w = *reinterpret_cast<const uint4*>(static_cast<const uint8_t*>(kv ? pg.v : pg.k) + from);
          const uint32_t ws[4] = {w.x, w.y, w.z, w.w};
          uint32_t* to = reinterpret_cast<uint32_t*>(u);
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const float2 lo = e4m3x2_to_float2(static_cast<uint16_t>(ws[i])), hi = e4m3x2_to_float2(static_cast<uint16_t>(ws[i] >> 16));
            to[2 * i] = pack_bf16x2(lo.x * f, lo.y * f);
            to[2 * i + 1] = pack_bf16x2(hi.x * f, hi.y * f);
          }
        } else {
          const uint4* w = reinterpret_cast<const uint4*>(static_cast<const __nv_bfloat16*>(kv ? pg.v : pg.k) + from);
          u[0] = w[0];
          u[1] = w[1];
        }
      }
      uint4* to = reinterpret_cast<uint4*>((kv ? v : k) + ((static_cast<long long>(b) * pg.most + j) * pg.Hkv + g) * DH + c);
      to[0] = u[0];
      to[1] = u[1];
    }
  }
}

// Up to 64 rows. 8 sequences of 4000 positions, 8 key heads of 128, 32 rows: 50 us, where the gather alone has 131 MB to write and to read again.
static bool is_step(const MdbPagedAttnArgs& a) { return static_cast<long long>(a.Sq) * (a.H / a.pages.Hkv) <= 64; }
static long long gathered(const MdbPagedAttnArgs& a) { return static_cast<long long>(a.pages.B) * a.pages.most * a.pages.Hkv * a.pages.Dh; }      // values

template <int DH, bool E4M3>
static int launch_gathered(const MdbPagedAttnArgs& a, cudaStream_t st) {
  const MdbPages& p = a.pages;
  __nv_bfloat16* k = reinterpret_cast<__nv_bfloat16*>(a.ws);
  __nv_bfloat16* v = k + gathered(a);
  int* lengths = reinterpret_cast<int*>(v + gathered(a));
  const long long blocks = (static_cast<long long>(p.most) * p.Hkv * (DH / 16) + 255) / 256;
  paged_gather_kernel<DH, E4M3><<<dim3(static_cast<unsigned>(std::min(blocks, 8ll * device_sm_count())), p.B), 256, 0, st>>>(a, k, v, lengths);
  if (cudaError_t e = cudaGetLastError(); e != cudaSuccess) return static_cast<int>(e);
  MdbTextAttnArgs t;
  memset(&t, 0, sizeof(t));
  t.q = a.q; t.k = k; t.v = v; t.o = a.o;
  t.kv_len = lengths; t.q_start_ptr = lengths + p.B;
  for (int i = 0; i < 3; ++i) {
    t.q_strides[i] = a.q_strides[i];
    t.o_strides[i] = a.o_strides[i];
  }
  t.k_strides[2] = t.v_strides[2] = DH;
  t.k_strides[1] = t.v_strides[1] = static_cast<long long>(p.Hkv) * DH;
  t.k_strides[0] = t.v_strides[0] = static_cast<long long>(p.most) * p.Hkv * DH;
  t.B = p.B; t.H = a.H; t.Hkv = p.Hkv; t.Sq = a.Sq; t.Skv = p.most; t.Dh = DH;
  t.window = 1 << 30;
  t.scale = a.scale;
  t.status = p.status;
  return mdb_text_attention_fwd(&t, st);
}

}  // namespace mdb

extern "C" long long mdb_paged_attention_floats(const MdbPagedAttnArgs* a) {
  if (a->pages.most == 0) return 0;
  if (!mdb::is_step(*a)) return mdb::gathered(*a) + 2ll * a->pages.B;
  if (mdb::is_whole(*a)) return 0;
  return 2ll * mdb::step_ctas(*a) * mdb::step_rows(*a) * (a->pages.Dh + 2);
}
extern "C" int mdb_paged_attention(const MdbPagedAttnArgs* a, cudaStream_t st) {
  const MdbPages& p = a->pages;
  if (p.B <= 0 || a->Sq <= 0 || p.Hkv <= 0 || p.most <= 0 || a->H % p.Hkv != 0 || (p.P != 16 && p.P != 32 && p.P != 64 && p.P != 128) || (p.Dh != 64 && p.Dh != 128)) return -1;
  const bool e4m3 = p.k_scale != nullptr;
  if (!mdb::is_step(*a)) {
    if (p.Dh == 128) return e4m3 ? mdb::launch_gathered<128, true>(*a, st) : mdb::launch_gathered<128, false>(*a, st);
    return e4m3 ? mdb::launch_gathered<64, true>(*a, st) : mdb::launch_gathered<64, false>(*a, st);
  }
  if (p.Dh == 128) return e4m3 ? mdb::launch_paged<128, true>(*a, st) : mdb::launch_paged<128, false>(*a, st);
  return e4m3 ? mdb::launch_paged<64, true>(*a, st) : mdb::launch_paged<64, false>(*a, st);
}

MDB_DEFINE_WAIT_LIMIT_SETTER(mdb_set_wait_limit_paged)
