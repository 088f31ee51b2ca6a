// New tokens of several sequences into the pages of their caches:
//
//   y = x rsqrt(mean(x^2) + eps) w  (q and k, where they have a weight);  (a, b) -> (a cos - b sin, b cos + a sin), a and b the halves of a head
//   keys and values go to the pages, rounded once to bf16 or to e4m3 in units of the page's scale; queries to an output, rounded to bf16
//
// The scale of a page and head follows from the largest value of the tokens that go there and is never smaller than the page's scale before, if the sequence
// had tokens in it. All of a head's tokens in a page belong to one block of threads, so that the scale is known before the first value is
// rounded, what was there is brought to it by the same block, and every element has one writer.
//
// What bounds it: memory, and the latency of its loads. 11.3 thousand tokens of sixteen prompts, 32 / 8 heads of 128, e4m3: 53 us a pass, 4.9 TB/s of what has to move (0.75 of the
// measured rate; 32 warps to an SM, issue slots 48 %). With 80 registers and 24 warps 63.5 us instead of 62.3, with four heads held in fp32 (168 registers) 178.
// At 64 registers, with which 32 warps fit, the forms of one or two rows to a group spill 100 to 244 bytes: the queries' path, with two rows and their angles, and the keys' share them.
// A token of each of 128 sequences: 7 us.
//
// A row (one head of one token) is held by Dh / 16 lanes, each with 8 values of either half: the halves of a rotated pair meet in one thread, the sum of squares takes
// two or three shuffles, and loads and stores are 16 bytes a lane.
#include "paged.cuh"

#include <algorithm>

namespace mdb {

constexpr int PA_THREADS = 256;

template <int DH> struct AppendRow {
  static constexpr int LANES = DH / 16;
  float2 x[2][4];      // of either half

  __device__ __forceinline__ static void fetch(uint4 (&u)[2], const __nv_bfloat16* row, int l) {
    u[0] = *reinterpret_cast<const uint4*>(row + l * 8);
    u[1] = *reinterpret_cast<const uint4*>(row + DH / 2 + l * 8);
  }
  __device__ __forceinline__ void set(const uint4 (&u)[2]) {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      x[h][0] = unpack_bf16x2(u[h].x);
      x[h][1] = unpack_bf16x2(u[h].y);
      x[h][2] = unpack_bf16x2(u[h].z);
      x[h][3] = unpack_bf16x2(u[h].w);
    }
  }
  __device__ __forceinline__ void clear() {
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
      for (int e = 0; e < 4; ++e) x[h][e] = make_float2(0.f, 0.f);
  }
  // 1 / sqrt(mean of the squares + eps); by whole warps: the lanes of a row add up theirs
  __device__ __forceinline__ float norm(float eps) const {
    float2 s = make_float2(0.f, 0.f);
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
      for (int e = 0; e < 4; ++e) s = ffma2(x[h][e], x[h][e], s);
    float t = s.x + s.y;
#pragma unroll
    for (int m = LANES / 2; m > 0; m >>= 1) t += __shfl_xor_sync(0xffffffffu, t, m);
    return rsqrtf(t * (1.f / DH) + eps);
  }
  __device__ __forceinline__ void weigh(const void* w, int f32, float r, int l) {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int d = h * (DH / 2) + l * 8;
      float2 f[4];
      if (f32) {
#pragma unroll
        for (int e = 0; e < 4; ++e) f[e] = reinterpret_cast<const float2*>(static_cast<const float*>(w) + d)[e];
      } else {
        const uint4 u = *reinterpret_cast<const uint4*>(static_cast<const __nv_bfloat16*>(w) + d);
        f[0] = unpack_bf16x2(u.x);
        f[1] = unpack_bf16x2(u.y);
        f[2] = unpack_bf16x2(u.z);
        f[3] = unpack_bf16x2(u.w);
      }
#pragma unroll
      for (int e = 0; e < 4; ++e) x[h][e] = fmul2(fmul2(x[h][e], make_float2(r, r)), f[e]);
    }
  }
  // products and sums are rounded one by one, as separate operations round them
  __device__ __forceinline__ void rotate(const AppendRow& angles) {      // cosines and sines
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const float2 a = x[0][e], b = x[1][e], c = angles.x[0][e], s = angles.x[1][e];
      const float2 bs = fmul2(b, s);
      x[0][e] = fadd2(fmul2(a, c), make_float2(-bs.x, -bs.y));
      x[1][e] = fadd2(fmul2(b, c), fmul2(a, s));
    }
  }
  __device__ __forceinline__ void set_angles(const float* cos, const float* sin, int l) {
#pragma unroll
    for (int e = 0; e < 4; e += 2) {
      *reinterpret_cast<float4*>(&x[0][e]) = *reinterpret_cast<const float4*>(cos + l * 8 + 2 * e);
      *reinterpret_cast<float4*>(&x[1][e]) = *reinterpret_cast<const float4*>(sin + l * 8 + 2 * e);
    }
  }
  // the largest size, infinity among them, NaN not
  __device__ __forceinline__ float most() const {
    float m = 0.f;
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
      for (int e = 0; e < 4; ++e) m = fmax3(m, fabsf(x[h][e].x), fabsf(x[h][e].y));
    return m;
  }
  __device__ __forceinline__ void infinite_to_nan() {
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        if (fabsf(x[h][e].x) == INFINITY) x[h][e].x = NAN;
        if (fabsf(x[h][e].y) == INFINITY) x[h][e].y = NAN;
      }
  }
  __device__ __forceinline__ void store_bf16(__nv_bfloat16* row, int l) const {
#pragma unroll
    for (int h = 0; h < 2; ++h)
      *reinterpret_cast<uint4*>(row + h * (DH / 2) + l * 8) = make_uint4(pack_bf16x2(x[h][0].x, x[h][0].y), pack_bf16x2(x[h][1].x, x[h][1].y),
                                                                         pack_bf16x2(x[h][2].x, x[h][2].y), pack_bf16x2(x[h][3].x, x[h][3].y));
  }
  __device__ __forceinline__ void store_e4m3(uint8_t* row, int l, float f) const {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      uint32_t w[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) w[e] = pack_e4m3x2(fmul2(x[h][e], make_float2(f, f)));
      *reinterpret_cast<uint2*>(row + h * (DH / 2) + l * 8) = make_uint2(w[0] | w[1] << 16, w[2] | w[3] << 16);
    }
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
      w[e] = pack_e4m3x2(make_float2(lo.x * f, lo.y * f)) | pack_e4m3x2(make_float2(hi.x * f, hi.y * f)) << 16;
    }
    *reinterpret_cast<uint4*>(at + i) = u;
  }
}

// A unit of work: the rows [row, row + count) of sequence b, which go to one page from `slot` on. count 0: nothing
struct AppendUnit {
  int b, index, slot, count, position;
  long long row;
};
// Sequences are disjoint and lie within the T rows whatever cu says: where it falls the largest end so far counts, and none passes the last one.
__device__ __forceinline__ int row_within(const MdbPagedAppendArgs& a, int b) { return min(max(a.cu[b], 0), static_cast<int>(a.T)); }
// By a whole warp: units are numbered sequence after sequence, a page after the other
__device__ __forceinline__ AppendUnit find_unit(const MdbPagedAppendArgs& a, int unit) {
  const int lane = threadIdx.x & 31, P = a.pages.P, shift = a.pages.shift, last = row_within(a, a.pages.B);
  AppendUnit u = {0, 0, 0, 0, 0, 0};
  int before = 0, largest = 0;
  bool fell = false;
  for (int b0 = 0; b0 < a.pages.B; b0 += 32) {
    int lo = 0, hi = 0, start = 0;
    if (b0 + lane < a.pages.B) {
      lo = row_within(a, b0 + lane);
      hi = row_within(a, b0 + lane + 1);
      start = a.start[b0 + lane];
      if (start < 0 || start > 1 << 30) start = 1 << 30;      // behind every page: reported like any position without one
    }
    fell = fell || __any_sync(0xffffffffu, hi < lo);
    if (fell) {
#pragma unroll
      for (int m = 1; m < 32; m <<= 1) {
        const int other = __shfl_up_sync(0xffffffffu, lo, m);
        if (lane >= m) lo = max(lo, other);
      }
      lo = max(lo, largest);
      hi = max(hi, lo);
    }
    largest = __reduce_max_sync(0xffffffffu, hi);
    int first = min(lo, last), length = min(hi, last) - first;
    const int mine = length > 0 ? ((start + length - 1) >> shift) - (start >> shift) + 1 : 0;
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
      u.index = (start >> shift) + j;
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
// By one block: ends that fall or lie outside the rows
__device__ __forceinline__ void check_ends(const MdbPagedAppendArgs& a) {
  for (int b = threadIdx.x; b < a.pages.B; b += PA_THREADS)
    if (a.cu[b] < 0 || a.cu[b] > a.cu[b + 1] || a.cu[b + 1] > a.T) report_status(a.pages.status, STATUS_BOUNDS, 186, b);
}

// Heads h0 .. hn - 1 of the rows before the first sequence and behind the last one come out as zeros; by the blocks from `units` on
template <int DH> __device__ __forceinline__ void clear_rows_of_none(const MdbPagedAppendArgs& a, int units, __nv_bfloat16* to, int heads, int h0, int hn) {
  using Row = AppendRow<DH>;
  constexpr int GROUPS = PA_THREADS / Row::LANES;
  const long long end = row_within(a, a.pages.B), first = min(static_cast<long long>(row_within(a, 0)), end);
  Row r;
  r.clear();
  for (long long i = (static_cast<long long>(blockIdx.x) - units) * GROUPS + threadIdx.x / Row::LANES; i < first + a.T - end; i += static_cast<long long>(gridDim.x - units) * GROUPS) {
    const long long t = i < first ? i : i - first + end;
    for (int h = h0; h < hn; ++h) r.store_bf16(to + (t * heads + h) * DH, threadIdx.x % Row::LANES);
  }
}

// grid: units, then rows of no sequence; parts of the heads: of the queries, of the keys, of the values. Finding the unit and its page takes as long as a
// few heads, so a block has several of them. Queries are turned one row of a group of lanes after the other, two heads at a time; of keys and values a block needs a head's rows
// of the whole unit at once, for its scale. Where a page has fewer rows than the block has groups of lanes, the groups share out the heads
// (TEAMS; 11.3 thousand tokens in pages of 16, e4m3: 28 / 4 heads of 64 61 -> 39 us, 32 / 8 of 128 92 -> 76; its registers would cost larger pages a tenth).
struct AppendGrid {
  int units, q_heads, kv_heads;      // heads of a block
};
template <int DH, bool E4M3, int ITERS, bool TEAMS>
__global__ void __launch_bounds__(PA_THREADS, ITERS == 4 ? 2 : 4)
paged_append_kernel(const __grid_constant__ MdbPagedAppendArgs a, const AppendGrid grid) {
  using Row = AppendRow<DH>;
  constexpr int LANES = Row::LANES, GROUPS = PA_THREADS / LANES;
  __shared__ float tops[2][PA_THREADS / 32];
  const int l = threadIdx.x % LANES, group = threadIdx.x / LANES, G = a.pages.Hkv;
  const int page_rows = TEAMS ? a.pages.P : GROUPS, teams = TEAMS ? GROUPS >> a.pages.shift : 1, team = TEAMS ? group >> a.pages.shift : 0, row = TEAMS ? group & (a.pages.P - 1) : group;      // a team is whole warps
  if (blockIdx.x == gridDim.x - 1 && blockIdx.y == 0) check_ends(a);      // behind the units
  const int q_parts = a.q != nullptr ? (a.H + grid.q_heads - 1) / grid.q_heads : 0, kv_parts = (G + grid.kv_heads - 1) / grid.kv_heads;
  if (static_cast<int>(blockIdx.y) < q_parts) {
    const int h0 = blockIdx.y * grid.q_heads, hn = min(a.H, h0 + grid.q_heads);
    if (static_cast<int>(blockIdx.x) >= grid.units) {      // queries behind the last sequence come out as zeros
      clear_rows_of_none<DH>(a, grid.units, static_cast<__nv_bfloat16*>(a.q_out), a.H, h0, hn);
      return;
    }
    const AppendUnit u = find_unit(a, blockIdx.x);
    const bool page = u.count > 0 && page_of(a.pages, u.b, u.index) >= 0;
    const int turned = page ? min(u.count, max(a.positions - u.position, 0)) : 0;      // rows that have a place and angles
    for (int t0 = 0; t0 < u.count; t0 += page_rows) {
      const int t = t0 + row;
      const bool in = t < u.count, placed = t < turned;
      const __nv_bfloat16* from = static_cast<const __nv_bfloat16*>(a.q) + (u.row + t) * a.q_strides[0];
      __nv_bfloat16* to = static_cast<__nv_bfloat16*>(a.q_out) + (u.row + t) * a.H * DH;
      Row angles;
      if (placed) angles.set_angles(a.cos + (u.position + t) * static_cast<long long>(DH / 2), a.sin + (u.position + t) * static_cast<long long>(DH / 2), l);
      for (int h = h0 + 2 * team; h < hn; h += 2 * teams) {
        uint4 raw[2][2];
        const bool two = h + 1 < hn;
        if (in) Row::fetch(raw[0], from + h * a.q_strides[1], l);
        if (in && two) Row::fetch(raw[1], from + (h + 1) * a.q_strides[1], l);
#pragma unroll
        for (int y = 0; y < 2; ++y) {
          if (y == 1 && !two) break;
          Row r;
          r.set(raw[y]);
          if (a.q_norm != nullptr) r.weigh(a.q_norm, a.q_norm_f32, r.norm(a.eps), l);
          if (placed) r.rotate(angles);
          else r.clear();
          if (in) r.store_bf16(to + (h + y) * DH, l);
        }
      }
    }
    return;
  }
  const int kv = static_cast<int>(blockIdx.y) >= q_parts + kv_parts, part = blockIdx.y - q_parts - kv * kv_parts;
  const int h0 = part * grid.kv_heads, hn = min(G, h0 + grid.kv_heads);
  __nv_bfloat16* k_out = kv == 0 ? static_cast<__nv_bfloat16*>(a.k_out) : nullptr;
  if (static_cast<int>(blockIdx.x) >= grid.units) {
    if (k_out != nullptr) clear_rows_of_none<DH>(a, grid.units, k_out, G, h0, hn);
    return;
  }
  const AppendUnit u = find_unit(a, blockIdx.x);
  if (u.count == 0) return;
  const int page = page_of(a.pages, u.b, u.index), turned = page >= 0 ? min(u.count, max(a.positions - u.position, 0)) : 0;
  if (turned < u.count && kv == 0 && part == 0 && threadIdx.x == 0) report_status(a.pages.status, STATUS_BOUNDS, 181, u.b);
  if (turned == 0 && k_out == nullptr) return;
  const long long* fs = kv ? a.v_strides : a.k_strides;
  const long long* ps = kv ? a.pages.v_strides : a.pages.k_strides;
  const __nv_bfloat16* from = static_cast<const __nv_bfloat16*>(kv ? a.v : a.k) + u.row * fs[0];
  const long long at = page * ps[0] + u.slot * DH;
  const int threads = page_rows * LANES, warps = threads / 32;      // of a team
#pragma unroll 1
  for (int turn = 0; h0 + turn * teams < hn; ++turn) {
    const int h = h0 + turn * teams + team;
    const bool mine = h < hn;
    unsigned char* scale = E4M3 && mine && page >= 0 ? (kv ? a.pages.v_scale : a.pages.k_scale) + page * a.pages.scale_strides[kv] + h : nullptr;
    const int before = scale != nullptr && u.slot > 0 ? min(static_cast<int>(*scale), 253) : 0;
    Row r[ITERS];
    uint4 raw[ITERS][2];
#pragma unroll
    for (int n = 0; n < ITERS; ++n)
      if (mine && n * page_rows + row < turned) Row::fetch(raw[n], from + (n * page_rows + row) * fs[0] + h * fs[1], l);
    float top = 0.f;
#pragma unroll
    for (int n = 0; n < ITERS; ++n) {
      const int t = n * page_rows + row;
      r[n].set(raw[n]);
      if (kv == 0 && a.k_norm != nullptr) r[n].weigh(a.k_norm, a.k_norm_f32, r[n].norm(a.eps), l);
      if (!mine || t >= turned) {
        r[n].clear();
        if (k_out != nullptr && mine && t < u.count) r[n].store_bf16(k_out + ((u.row + t) * G + h) * DH, l);
        continue;
      }
      if (kv == 0) {
        Row angles;
        angles.set_angles(a.cos + (u.position + t) * static_cast<long long>(DH / 2), a.sin + (u.position + t) * static_cast<long long>(DH / 2), l);
        r[n].rotate(angles);
        if (k_out != nullptr) r[n].store_bf16(k_out + ((u.row + t) * G + h) * DH, l);
      }
      if (!E4M3) {
        r[n].store_bf16(static_cast<__nv_bfloat16*>(kv ? a.pages.v : a.pages.k) + at + h * ps[1] + t * DH, l);
      } else {
        float size = r[n].most();
        if (size == INFINITY) {
          r[n].infinite_to_nan();
          size = r[n].most();
        }
        top = fmaxf(top, size);
      }
    }
    if (!E4M3 || turned == 0) continue;
#pragma unroll
    for (int m = 16; m > 0; m >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, m));
    if ((threadIdx.x & 31) == 0) tops[turn & 1][threadIdx.x >> 5] = top;
    __syncthreads();      // a turn's half of `tops` is written again behind the next one's barrier
    if (!mine) continue;
    for (int i = 0; i < warps; ++i) top = fmaxf(top, tops[turn & 1][team * warps + i]);
    const int byte = max(scale_byte(top), before), thread = threadIdx.x - team * threads;
    uint8_t* to = static_cast<uint8_t*>(kv ? a.pages.v : a.pages.k) + at + h * ps[1];
    if (u.slot > 0 && byte > before) rescale(to - u.slot * DH, u.slot * DH, byte - before, thread, threads);
    const float f = scale_inverse(byte);
#pragma unroll
    for (int n = 0; n < ITERS; ++n)
      if (n * page_rows + row < turned) r[n].store_e4m3(to + (n * page_rows + row) * DH, l, f);
    if (thread == 0 && byte != before) *scale = static_cast<unsigned char>(byte);
  }
}

// A row for each sequence: no page gets a second one, so a row's lanes know its scale by themselves, and heads, keys and values of all sequences are one line of
// rows. What bounds it is the way from the length to the page, its scale and the value; a block for each page and head took 22 us for 128 tokens of 32 / 8 heads.
constexpr int PT_THREADS = 128;
template <int DH, bool E4M3>
__global__ void __launch_bounds__(PT_THREADS)
paged_append_token_kernel(const __grid_constant__ MdbPagedAppendArgs a) {
  using Row = AppendRow<DH>;
  constexpr int LANES = Row::LANES;
  const int l = threadIdx.x % LANES, H = a.q != nullptr ? a.H : 0, heads = H + 2 * a.pages.Hkv;
  const long long n = (blockIdx.x * static_cast<long long>(PT_THREADS) + threadIdx.x) / LANES;
  const bool in = n < static_cast<long long>(a.pages.B) * heads;
  const int b = in ? static_cast<int>(n / heads) : 0, h = in ? static_cast<int>(n - static_cast<long long>(b) * heads) : 0;
  const bool is_q = h < H, is_v = h >= H + a.pages.Hkv;
  const int g = is_q ? h : is_v ? h - H - a.pages.Hkv : h - H;
  const int p = a.start[b];
  Row r;
  uint4 raw[2];
  if (in) Row::fetch(raw, is_q ? static_cast<const __nv_bfloat16*>(a.q) + b * a.q_strides[0] + g * a.q_strides[1]
                      : is_v ? static_cast<const __nv_bfloat16*>(a.v) + b * a.v_strides[0] + g * a.v_strides[1] : static_cast<const __nv_bfloat16*>(a.k) + b * a.k_strides[0] + g * a.k_strides[1], l);
  const int page = p >= 0 && p < a.positions ? page_of(a.pages, b, p >> a.pages.shift) : -1, slot = p & (a.pages.P - 1);
  unsigned char* scale = E4M3 && page >= 0 && !is_q ? (is_v ? a.pages.v_scale : a.pages.k_scale) + page * a.pages.scale_strides[is_v] + g : nullptr;
  const int before = scale != nullptr && slot > 0 ? min(static_cast<int>(*scale), 253) : 0;
  const void* w = is_q ? a.q_norm : is_v ? nullptr : a.k_norm;
  r.set(raw);
  if (a.q_norm != nullptr || a.k_norm != nullptr) {      // by whole warps, whose rows may be of several kinds
    const float f = r.norm(a.eps);
    if (w != nullptr) r.weigh(w, is_q ? a.q_norm_f32 : a.k_norm_f32, f, l);
  }
  if (!in) return;
  if (page >= 0 && !is_v) {
    Row angles;
    angles.set_angles(a.cos + p * static_cast<long long>(DH / 2), a.sin + p * static_cast<long long>(DH / 2), l);
    r.rotate(angles);
  }
  if (is_q) {
    if (page < 0) r.clear();
    r.store_bf16(static_cast<__nv_bfloat16*>(a.q_out) + (static_cast<long long>(b) * a.H + h) * DH, l);
    return;
  }
  if (page < 0) r.clear();
  if (!is_v && a.k_out != nullptr) r.store_bf16(static_cast<__nv_bfloat16*>(a.k_out) + (static_cast<long long>(b) * a.pages.Hkv + g) * DH, l);
  if (page < 0) {
    if (l == 0) report_status(a.pages.status, STATUS_BOUNDS, 181, b);
    return;
  }
  const long long* ps = is_v ? a.pages.v_strides : a.pages.k_strides;
  const long long at = page * ps[0] + g * ps[1];
  void* pool = is_v ? a.pages.v : a.pages.k;
  if (!E4M3) {
    r.store_bf16(static_cast<__nv_bfloat16*>(pool) + at + slot * DH, l);
    return;
  }
  const uint32_t mine = ((1u << LANES) - 1) << ((threadIdx.x & 31) / LANES * LANES);
  float top = r.most();
  if (top == INFINITY) {
    r.infinite_to_nan();
    top = r.most();
  }
#pragma unroll
  for (int m = LANES / 2; m > 0; m >>= 1) top = fmaxf(top, __shfl_xor_sync(mine, top, m));
  const int byte = max(scale_byte(top), before);
  uint8_t* to = static_cast<uint8_t*>(pool) + at;
  if (slot > 0 && byte > before) rescale(to, slot * DH, byte - before, l, LANES);
  r.store_e4m3(to + slot * DH, l, scale_inverse(byte));
  if (l == 0 && byte != before) *scale = static_cast<unsigned char>(byte);
}

template <int DH, bool E4M3>
static int launch_append(const MdbPagedAppendArgs& a, cudaStream_t st) {
  if (a.cu == nullptr) {
    const long long rows = static_cast<long long>(a.pages.B) * ((a.q != nullptr ? a.H : 0) + 2 * a.pages.Hkv), per = PT_THREADS / AppendRow<DH>::LANES;
    paged_append_token_kernel<DH, E4M3><<<static_cast<unsigned>((rows + per - 1) / per), PT_THREADS, 0, st>>>(a);
    return static_cast<int>(cudaGetLastError());
  }
  // a sequence of n > 0 rows touches no more than (n - 1) / P + 2 pages, and no more than n
  const int B = a.pages.B, P = a.pages.P, groups = PA_THREADS / AppendRow<DH>::LANES;
  const long long units = std::min(a.T, a.T / P + 2ll * B);
  if (units > 0x7ffffff0) return -8;
  const int spare = a.q != nullptr || a.k_out != nullptr ? 8 : 1;      // blocks for rows of no sequence and a look at the ends
  const int rows = static_cast<int>(std::min<long long>(P, a.T)), H = a.q != nullptr ? a.H : 0, G = a.pages.Hkv;      // rows of a unit, at most
  // heads of a block: sixteen and four, fewer where that leaves fewer than six blocks to an SM (11.3 thousand tokens, 32 / 8 heads of 128: 59.4 us, with eight and two 62.3,
  // four and one 69.6; 4.2 thousand, 28 / 4 heads of 64, bf16 pages: eight and two 20.5 us, eight and one 22.5)
  AppendGrid grid = {static_cast<int>(units), 16, 4};
  const auto parts = [&]() { return (H + grid.q_heads - 1) / grid.q_heads + 2 * ((G + grid.kv_heads - 1) / grid.kv_heads); };
  while (grid.q_heads > 1 && units * parts() < 6ll * device_sm_count()) {
    grid.q_heads /= 2;
    grid.kv_heads = std::max(grid.kv_heads / 2, 1);
  }
  const dim3 blocks(static_cast<unsigned>(units) + spare, parts());
  if (P < groups) paged_append_kernel<DH, E4M3, 1, true><<<blocks, PA_THREADS, 0, st>>>(a, grid);
  else if (rows <= groups) paged_append_kernel<DH, E4M3, 1, false><<<blocks, PA_THREADS, 0, st>>>(a, grid);
  else if (rows <= 2 * groups) paged_append_kernel<DH, E4M3, 2, false><<<blocks, PA_THREADS, 0, st>>>(a, grid);
  else paged_append_kernel<DH, E4M3, 4, false><<<blocks, PA_THREADS, 0, st>>>(a, grid);
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
