// New tokens of several sequences into the pages of their caches:
//
//   y = x rsqrt(mean(x^2) + eps) w  (q and k, where they have a weight);  (a, b) -> (a cos - b sin, b cos + a sin), a and b the halves of a head
//   keys and values go to the pages, rounded once to bf16 or to e4m3 in units of the page's scale; queries to an output, rounded to bf16
//
// The scale of a page and head follows from the largest value of the tokens that go there and is never smaller than the page's scale before, if the sequence
// had tokens in it. All of a head's tokens in a page belong to one block of threads, so that the scale is known before the first value is
// rounded, what was there is brought to it by the same block, and every element has one writer.
//
// A row (one head of one token) is held by Dh / 16 lanes, each with 8 values of either half: the halves of a rotated pair meet in one thread, the sum of squares takes
// two or three shuffles, and loads and stores are 16 bytes a lane.
#include "paged.cuh"

#include <algorithm>

namespace mdb {

constexpr int PA_THREADS = 256;

template <int DH> struct AppendRow {
  static constexpr int LANES = DH / 16;
  float x[16];

  __device__ __forceinline__ void load(const __nv_bfloat16* row, int l) {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const uint4 u = *reinterpret_cast<const uint4*>(row + h * (DH / 2) + l * 8);
      const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float2 f = unpack_bf16x2(w[e]);
        x[h * 8 + 2 * e] = f.x;
        x[h * 8 + 2 * e + 1] = f.y;
      }
    }
  }
  __device__ __forceinline__ static float sum(float s) {
#pragma unroll
    for (int m = LANES / 2; m > 0; m >>= 1) s += __shfl_xor_sync(0xffffffffu, s, m);
    return s;
  }
  // by whole warps: the lanes of a row add up their squares
  __device__ __forceinline__ void norm(const void* w, int f32, float eps, int l) {
    float s = 0.f;
#pragma unroll
    for (int e = 0; e < 16; ++e) s = fmaf(x[e], x[e], s);
    const float r = rsqrtf(sum(s) * (1.f / DH) + eps);
#pragma unroll
    for (int e = 0; e < 16; ++e) {
      const int d = (e >> 3) * (DH / 2) + l * 8 + (e & 7);
      x[e] = x[e] * r * (f32 ? static_cast<const float*>(w)[d] : __bfloat162float(static_cast<const __nv_bfloat16*>(w)[d]));
    }
  }
  // products and sums are rounded one by one, as separate operations round them
  __device__ __forceinline__ void rotate(const float* cos, const float* sin, int l) {
    float c[8], s[8];
#pragma unroll
    for (int e = 0; e < 8; e += 4) {
      *reinterpret_cast<float4*>(c + e) = *reinterpret_cast<const float4*>(cos + l * 8 + e);
      *reinterpret_cast<float4*>(s + e) = *reinterpret_cast<const float4*>(sin + l * 8 + e);
    }
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const float a = x[e], b = x[e + 8];
      x[e] = __fsub_rn(__fmul_rn(a, c[e]), __fmul_rn(b, s[e]));
      x[e + 8] = __fadd_rn(__fmul_rn(b, c[e]), __fmul_rn(a, s[e]));
    }
  }
  __device__ __forceinline__ float most() const {      // of the finite values
    float m = 0.f;
#pragma unroll
    for (int e = 0; e < 16; ++e) {
      const float a = fabsf(x[e]);
      m = a < INFINITY ? fmaxf(m, a) : m;
    }
    return m;
  }
  __device__ __forceinline__ void store_bf16(__nv_bfloat16* row, int l) const {
#pragma unroll
    for (int h = 0; h < 2; ++h)
      *reinterpret_cast<uint4*>(row + h * (DH / 2) + l * 8) = make_uint4(pack_bf16x2(x[h * 8], x[h * 8 + 1]), pack_bf16x2(x[h * 8 + 2], x[h * 8 + 3]),
                                                                         pack_bf16x2(x[h * 8 + 4], x[h * 8 + 5]), pack_bf16x2(x[h * 8 + 6], x[h * 8 + 7]));
  }
  __device__ __forceinline__ void store_e4m3(uint8_t* row, int l, float f) const {
#pragma unroll
    for (int h = 0; h < 2; ++h)
      *reinterpret_cast<uint2*>(row + h * (DH / 2) + l * 8) = make_uint2(pack_e4m3x2(x[h * 8] * f, x[h * 8 + 1] * f) | pack_e4m3x2(x[h * 8 + 2] * f, x[h * 8 + 3] * f) << 16,
                                                                         pack_e4m3x2(x[h * 8 + 4] * f, x[h * 8 + 5] * f) | pack_e4m3x2(x[h * 8 + 6] * f, x[h * 8 + 7] * f) << 16);
  }
};

// `bytes` of a page (a multiple of 16) to a scale that is 2^by smaller values, by `threads` threads of which this one is `t`
__device__ __forceinline__ void rescale(uint8_t* at, int bytes, int by, int t, int threads) {
  const float f = scale_inverse(127 + min(by, 126));
  for (int i = t * 16; i < bytes; i += threads * 16) {
    uint4 u = *reinterpret_cast<uint4*>(at + i);
    uint32_t* w = reinterpret_cast<uint32_t*>(&u);
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const float2 lo = e4m3x2_to_float2(static_cast<uint16_t>(w[e])), hi = e4m3x2_to_float2(static_cast<uint16_t>(w[e] >> 16));
      w[e] = pack_e4m3x2(lo.x * f, lo.y * f) | pack_e4m3x2(hi.x * f, hi.y * f) << 16;
    }
    *reinterpret_cast<uint4*>(at + i) = u;
  }
}

// A unit of work: the rows [row, row + count) of sequence b, which go to one page from `slot` on. count 0: nothing
struct AppendUnit {
  int b, index, slot, count, position;
  long long row;
};
// The rows of sequence b; what the lengths say is held within the T rows
__device__ __forceinline__ void rows_of(const MdbPagedAppendArgs& a, int b, long long& first, int& length, int& start) {
  const long long lo = a.cu == nullptr ? b : min(max(static_cast<long long>(a.cu[b]), 0ll), a.T);
  const long long hi = a.cu == nullptr ? b + 1 : min(max(static_cast<long long>(a.cu[b + 1]), lo), a.T);
  first = lo;
  length = static_cast<int>(hi - lo);
  start = a.start[b];
  if (start < 0 || start > 1 << 30) start = 1 << 30;      // behind every page: reported like any position without one
}
// By a whole warp: units are numbered sequence after sequence, a page after the other
__device__ __forceinline__ AppendUnit find_unit(const MdbPagedAppendArgs& a, int unit) {
  const int lane = threadIdx.x & 31, P = a.pages.P;
  AppendUnit u = {0, 0, 0, 0, 0, 0};
  int before = 0;
  for (int b0 = 0; b0 < a.pages.B; b0 += 32) {
    long long first = 0;
    int length = 0, start = 0;
    if (b0 + lane < a.pages.B) rows_of(a, b0 + lane, first, length, start);
    const int mine = length > 0 ? (start + length - 1) / P - start / P + 1 : 0;
    int upto = mine;
#pragma unroll
    for (int m = 1; m < 32; m <<= 1) {
      const int other = __shfl_up_sync(0xffffffffu, upto, m);
      if (lane >= m) upto += other;
    }
    const uint32_t behind = __ballot_sync(0xffffffffu, before + upto > unit);
    if (behind != 0) {
      const int at = __ffs(behind) - 1;
      first = __shfl_sync(0xffffffffu, first, at);
      length = __shfl_sync(0xffffffffu, length, at);
      start = __shfl_sync(0xffffffffu, start, at);
      const int j = unit - before - __shfl_sync(0xffffffffu, upto - mine, at);
      u.b = b0 + at;
      u.index = start / P + j;
      const int from = max(u.index * P, start), to = static_cast<int>(min(static_cast<long long>(u.index + 1) * P, static_cast<long long>(start) + length));
      u.slot = from - u.index * P;
      u.count = to - from;
      u.position = from;
      u.row = first + (from - start);
      return u;
    }
    before += __shfl_sync(0xffffffffu, upto, 31);
  }
  return u;
}

// grid: units, then rows behind the last sequence; key heads; keys, values, queries of the head's group
template <int DH, bool E4M3, int ITERS>
__global__ void __launch_bounds__(PA_THREADS)
paged_append_kernel(const __grid_constant__ MdbPagedAppendArgs a, const int units) {
  using Row = AppendRow<DH>;
  constexpr int LANES = Row::LANES, GROUPS = PA_THREADS / LANES;
  __shared__ float tops[PA_THREADS / 32];
  const int l = threadIdx.x % LANES, group = threadIdx.x / LANES, g = blockIdx.y, kind = blockIdx.z;
  const int rep = a.q != nullptr ? a.H / a.pages.Hkv : 0;
  if (static_cast<int>(blockIdx.x) >= units) {      // queries behind the last sequence come out as zeros
    if (kind != 2) return;
    const long long end = min(max(static_cast<long long>(a.cu[a.pages.B]), 0ll), a.T);
    for (long long i = (static_cast<long long>(blockIdx.x) - units) * GROUPS + group; i < (a.T - end) * rep; i += static_cast<long long>(gridDim.x - units) * GROUPS) {
      __nv_bfloat16* to = static_cast<__nv_bfloat16*>(a.q_out) + ((end + i / rep) * a.H + g * rep + i % rep) * DH;
#pragma unroll
      for (int h = 0; h < 2; ++h) *reinterpret_cast<uint4*>(to + h * (DH / 2) + l * 8) = make_uint4(0, 0, 0, 0);
    }
    return;
  }
  const AppendUnit u = find_unit(a, blockIdx.x);
  if (u.count == 0) return;
  const int page = page_of(a.pages, u.b, u.index), placed = page >= 0 ? min(u.count, max(a.positions - u.position, 0)) : 0;
  if (placed < u.count && threadIdx.x == 0) report_status(a.pages.status, STATUS_BOUNDS, 181, u.b);
  if (kind == 2) {
    for (int i0 = 0; i0 < u.count * rep; i0 += GROUPS) {
      const int i = i0 + group, t = i / rep, h = g * rep + i % rep;
      const bool in = i < u.count * rep && t < placed;
      Row r;
      if (in) r.load(static_cast<const __nv_bfloat16*>(a.q) + (u.row + t) * a.q_strides[0] + h * a.q_strides[1], l);
      if (a.q_norm != nullptr) r.norm(a.q_norm, a.q_norm_f32, a.eps, l);
      if (in) r.rotate(a.cos + (u.position + t) * static_cast<long long>(DH / 2), a.sin + (u.position + t) * static_cast<long long>(DH / 2), l);
      if (i < u.count * rep && !in) {
#pragma unroll
        for (int e = 0; e < 16; ++e) r.x[e] = 0.f;
      }
      if (i < u.count * rep) r.store_bf16(static_cast<__nv_bfloat16*>(a.q_out) + ((u.row + t) * a.H + h) * DH, l);
    }
    return;
  }
  if (placed == 0) return;
  const __nv_bfloat16* from = static_cast<const __nv_bfloat16*>(kind ? a.v : a.k);
  const long long* fs = kind ? a.v_strides : a.k_strides;
  const long long* ps = kind ? a.pages.v_strides : a.pages.k_strides;
  const long long at = page * ps[0] + g * ps[1];
  Row r[ITERS];
  float top = 0.f;
#pragma unroll
  for (int n = 0; n < ITERS; ++n) {
    const int t = n * GROUPS + group;
    if (t < placed) r[n].load(from + (u.row + t) * fs[0] + g * fs[1], l);
    if (kind == 0 && a.k_norm != nullptr) r[n].norm(a.k_norm, a.k_norm_f32, a.eps, l);
    if (t < placed) {
      if (kind == 0) r[n].rotate(a.cos + (u.position + t) * static_cast<long long>(DH / 2), a.sin + (u.position + t) * static_cast<long long>(DH / 2), l);
      if (E4M3) top = fmaxf(top, r[n].most());
      else r[n].store_bf16(static_cast<__nv_bfloat16*>(kind ? a.pages.v : a.pages.k) + at + (u.slot + t) * DH, l);
    }
  }
  if (!E4M3) return;
#pragma unroll
  for (int m = 16; m > 0; m >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, m));
  if ((threadIdx.x & 31) == 0) tops[threadIdx.x >> 5] = top;
  unsigned char* scale = (kind ? a.pages.v_scale : a.pages.k_scale) + page * a.pages.scale_strides[kind] + g;
  const int before = u.slot > 0 ? min(static_cast<int>(*scale), 253) : 0;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < PA_THREADS / 32; ++w) top = fmaxf(top, tops[w]);
  const int byte = max(scale_byte(top), before);
  uint8_t* to = static_cast<uint8_t*>(kind ? a.pages.v : a.pages.k) + at;
  if (u.slot > 0 && byte > before) rescale(to, u.slot * DH, byte - before, threadIdx.x, PA_THREADS);
  const float f = scale_inverse(byte);
#pragma unroll
  for (int n = 0; n < ITERS; ++n) {
    const int t = n * GROUPS + group;
    if (t < placed) r[n].store_e4m3(to + (u.slot + t) * DH, l, f);
  }
  if (threadIdx.x == 0) *scale = static_cast<unsigned char>(byte);
}

template <int DH, bool E4M3>
static int launch_append(const MdbPagedAppendArgs& a, cudaStream_t st) {
  // a sequence of n > 0 rows touches no more than (n - 1) / P + 2 pages, and no more than n
  const int B = a.pages.B, P = a.pages.P, groups = PA_THREADS / AppendRow<DH>::LANES;
  const long long units = a.cu == nullptr ? B : std::min(a.T, a.T / P + 2ll * B);
  if (units > 0x7ffffff0) return -8;
  const int spare = a.cu != nullptr && a.q != nullptr ? 8 : 0;      // blocks for rows behind the last sequence
  const dim3 grid(static_cast<unsigned>(units) + spare, a.pages.Hkv, a.q != nullptr ? 3 : 2);
  const int rows = a.cu == nullptr ? 1 : static_cast<int>(std::min<long long>(P, a.T));      // of a unit, at most
  if (rows <= groups) paged_append_kernel<DH, E4M3, 1><<<grid, PA_THREADS, 0, st>>>(a, static_cast<int>(units));
  else if (rows <= 2 * groups) paged_append_kernel<DH, E4M3, 2><<<grid, PA_THREADS, 0, st>>>(a, static_cast<int>(units));
  else paged_append_kernel<DH, E4M3, 4><<<grid, PA_THREADS, 0, st>>>(a, static_cast<int>(units));
  return static_cast<int>(cudaGetLastError());
}

}  // namespace mdb

extern "C" int mdb_paged_append(const MdbPagedAppendArgs* a, cudaStream_t st) {
  const MdbPages& p = a->pages;
  if (p.B <= 0 || a->T <= 0 || p.Hkv <= 0 || (p.P != 16 && p.P != 32 && p.P != 64 && p.P != 128)) return -1;
  if (p.Dh == 128) return p.k_scale != nullptr ? mdb::launch_append<128, true>(*a, st) : mdb::launch_append<128, false>(*a, st);
  if (p.Dh == 64) return p.k_scale != nullptr ? mdb::launch_append<64, true>(*a, st) : mdb::launch_append<64, false>(*a, st);
  return -2;
}
