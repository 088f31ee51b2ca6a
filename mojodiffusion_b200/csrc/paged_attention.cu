// Attention over the pages of several sequences: query row i of sequence b stands at position p = kv_len[b] - Sq + i and sees the keys up to p.
//
//   o_i = sum_j p_ij v_j / sum_j p_ij,  p_ij = exp(s_ij - max),  s_ij = scale 2^ek q_i . k_j;  values are in units of 2^ev; ek, ev of the page and head
//
// A block of threads per query row: groups of lanes take the keys in turn, each with its own reference and sums, which meet in shared memory.
#include "paged.cuh"

namespace mdb {

constexpr int PT_THREADS = 128;

// 16 neighbours of a key or a value
template <bool E4M3> __device__ __forceinline__ void load16(float (&x)[16], const void* base, long long at) {
  if (E4M3) {
    const uint4 u = *reinterpret_cast<const uint4*>(static_cast<const uint8_t*>(base) + at);
    const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const float2 lo = e4m3x2_to_float2(static_cast<uint16_t>(w[e])), hi = e4m3x2_to_float2(static_cast<uint16_t>(w[e] >> 16));
      x[4 * e] = lo.x; x[4 * e + 1] = lo.y; x[4 * e + 2] = hi.x; x[4 * e + 3] = hi.y;
    }
  } else {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const uint4 u = *reinterpret_cast<const uint4*>(static_cast<const __nv_bfloat16*>(base) + at + h * 8);
      const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float2 f = unpack_bf16x2(w[e]);
        x[h * 8 + 2 * e] = f.x;
        x[h * 8 + 2 * e + 1] = f.y;
      }
    }
  }
}

template <int DH, bool E4M3>
__global__ void __launch_bounds__(PT_THREADS) paged_rows_kernel(const __grid_constant__ MdbPagedAttnArgs a) {
  constexpr int LANES = DH / 16, GROUPS = PT_THREADS / LANES;
  __shared__ float part_m[GROUPS], part_l[GROUPS], part_o[GROUPS][DH];
  const MdbPages& p = a.pages;
  const int l = threadIdx.x % LANES, group = threadIdx.x / LANES;
  const int h = blockIdx.x % a.H, i = blockIdx.x / a.H, b = blockIdx.y, g = h / (a.H / p.Hkv);
  const int length = min(max(a.kv_len[b], 0), p.most), keys = max(length - a.Sq + i + 1, 0);
  float q[16], o[16], m = -INFINITY, sum = 0.f;
  load16<false>(q, a.q, b * a.q_strides[0] + i * a.q_strides[1] + h * a.q_strides[2] + l * 16);
#pragma unroll
  for (int e = 0; e < 16; ++e) o[e] = 0.f;
  for (int j0 = 0; j0 < keys; j0 += GROUPS) {
    const int j = j0 + group;
    const int page = j < keys ? page_of(p, b, j / p.P) : -1;
    if (page < 0 && j < keys) report_status(p.status, STATUS_BOUNDS, 182, b);
    float s = 0.f, x[16];
    if (page >= 0) {
      load16<E4M3>(x, p.k, page * p.k_strides[0] + g * p.k_strides[1] + (j % p.P) * DH + l * 16);
#pragma unroll
      for (int e = 0; e < 16; ++e) s = fmaf(q[e], x[e], s);
    }
#pragma unroll
    for (int n = LANES / 2; n > 0; n >>= 1) s += __shfl_xor_sync(0xffffffffu, s, n);
    if (page < 0) continue;
    s *= a.scale * 1.4426950408889634f;
    if (E4M3) s *= scale_value(p.k_scale[page * p.scale_strides[0] + g]);
    float top, w;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(top) : "f"(m), "f"(s));
    const float f = m == -INFINITY ? 0.f : exp2f(m - top);
    w = top == -INFINITY ? 0.f : exp2f(s - top);
    m = top;
    sum = sum * f + w;
    load16<E4M3>(x, p.v, page * p.v_strides[0] + g * p.v_strides[1] + (j % p.P) * DH + l * 16);
    if (E4M3) w *= scale_value(p.v_scale[page * p.scale_strides[1] + g]);
#pragma unroll
    for (int e = 0; e < 16; ++e) o[e] = o[e] * f + w * x[e];
  }
  if (l == 0) {
    part_m[group] = m;
    part_l[group] = sum;
  }
#pragma unroll
  for (int e = 0; e < 16; ++e) part_o[group][l * 16 + e] = o[e];
  __syncthreads();
  for (int d = threadIdx.x; d < DH; d += PT_THREADS) {
    float top = -INFINITY, total = 0.f, v = 0.f;
    for (int n = 0; n < GROUPS; ++n) asm("max.NaN.f32 %0, %1, %2;" : "=f"(top) : "f"(top), "f"(part_m[n]));
    for (int n = 0; n < GROUPS; ++n) {
      const float f = part_m[n] == -INFINITY ? 0.f : exp2f(part_m[n] - top);
      total += f * part_l[n];
      v += f * part_o[n][d];
    }
    static_cast<__nv_bfloat16*>(a.o)[b * a.o_strides[0] + i * a.o_strides[1] + h * a.o_strides[2] + d] = __float2bfloat16_rn(top == -INFINITY || total == 0.f ? 0.f : v / total);
  }
}

template <int DH, bool E4M3>
static int launch_paged(const MdbPagedAttnArgs& a, cudaStream_t st) {
  paged_rows_kernel<DH, E4M3><<<dim3(a.Sq * a.H, a.pages.B), PT_THREADS, 0, st>>>(a);
  return static_cast<int>(cudaGetLastError());
}

}  // namespace mdb

extern "C" int mdb_paged_attention(const MdbPagedAttnArgs* a, cudaStream_t st) {
  const MdbPages& p = a->pages;
  if (p.B <= 0 || a->Sq <= 0 || p.Hkv <= 0 || a->H % p.Hkv != 0 || (p.P != 16 && p.P != 32 && p.P != 64 && p.P != 128)) return -1;
  if (p.Dh == 128) return p.k_scale != nullptr ? mdb::launch_paged<128, true>(*a, st) : mdb::launch_paged<128, false>(*a, st);
  if (p.Dh == 64) return p.k_scale != nullptr ? mdb::launch_paged<64, true>(*a, st) : mdb::launch_paged<64, false>(*a, st);
  return -2;
}
