// What the kernels of the language models' attention share: which keys a query sees, and the bias of a relative position.
#pragma once
#include "common.cuh"
#include "kernels_api.h"

namespace mdb {

constexpr int TXT_FAR = 1 << 30;
constexpr float TXT_LOG2E = 1.4426950408889634f, TXT_LN2 = 0.6931471805599453f;

__device__ __forceinline__ float text_param(const void* p, int is_f32, long long i) {
  return is_f32 ? static_cast<const float*>(p)[i] : __bfloat162float(static_cast<const __nv_bfloat16*>(p)[i]);
}

// the keys of batch entry b end at `valid`, its query row 0 stands at position `start`
struct TextSight {
  int valid, start;
};
__device__ __forceinline__ TextSight text_sight(const MdbTextAttnArgs& a, int b) {
  TextSight s;
  s.valid = a.kv_len != nullptr ? min(max(a.kv_len[b], 0), a.Skv) : a.Skv;
  s.start = a.q_start_ptr != nullptr ? a.q_start_ptr[b] : a.q_start;
  s.start = min(max(s.start, -TXT_FAR), TXT_FAR - 1 - a.Sq);      // every position below TXT_FAR, which stands for no window
  return s;
}

// Keys that the queries at positions p_lo .. p_hi see together: [0, sinks) and [lo, end), lo >= sinks unless everything from 0 on is seen.
// Every query sees a subset; with BIAS (no mask but the length) each sees all of them.
struct TextKeys {
  int sinks, lo, end;
};
template <bool BIAS>
__device__ __forceinline__ TextKeys text_keys(const MdbTextAttnArgs& a, const TextSight& s, int p_lo, int p_hi) {
  TextKeys k;
  k.end = BIAS ? s.valid : max(min(p_hi + 1, s.valid), 0);
  k.lo = BIAS ? 0 : min(max(p_lo - a.window + 1, 0), k.end);
  k.sinks = BIAS ? 0 : min(a.sinks, k.end);
  if (k.sinks >= k.lo) k.sinks = k.lo = 0;
  return k;
}

// Packed sequences: a unit is a block of `gran` rows of one sequence. Units stand in the order of their blocks' numbers, the last blocks, which have the most keys, of all
// sequences first. Up to 32 sequences: a warp finds a unit from the lengths (a lane each); more: a kernel before has written down the units, sequence after sequence.
struct TextUnit {
  int base, rows, block;      // first row and length of the sequence; rows 0: no unit
};
// Ends are held within the rows. Where they fall there is no unit: sequences would have rows in common.
__device__ __forceinline__ int text_row_within(const MdbTextAttnArgs& a, int b) { return min(max(a.cu[b], 0), a.Sq); }
__device__ __forceinline__ TextUnit text_unit(const MdbTextAttnArgs& a, int unit, int gran) {
  if (a.units != nullptr) {
    const int4 u = a.units[unit];
    return {u.x, u.y, u.z};
  }
  const int lane = threadIdx.x & 31;
  const int first = lane < a.B ? text_row_within(a, lane) : 0;
  int rows = lane < a.B ? text_row_within(a, lane + 1) - first : 0;
  if (__any_sync(0xffffffffu, rows < 0)) rows = 0;
  const int n = (rows + gran - 1) / gran;
  const auto from = [&](int level) { return static_cast<int>(__reduce_add_sync(0xffffffffu, static_cast<unsigned>(max(n - level, 0)))); };      // blocks of this number or a larger one
  int lo = 0, hi = __reduce_max_sync(0xffffffffu, n);      // from(lo) > unit >= from(hi)
  if (unit >= from(0)) return {0, 0, 0};
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (from(mid) > unit) lo = mid;
    else hi = mid;
  }
  const uint32_t have = __ballot_sync(0xffffffffu, n > lo);
  const int rank = unit - from(lo + 1);
  const int at = __ffs(__ballot_sync(0xffffffffu, n > lo && __popc(have & ((1u << lane) - 1u)) == rank)) - 1;
  return {__shfl_sync(0xffffffffu, first, at), __shfl_sync(0xffffffffu, rows, at), lo};
}
// The same with the first rows, whose keys have the most queries, of all sequences first: the numbers of a sequence's blocks the other way round
__device__ __forceinline__ TextUnit text_unit_of_keys(const MdbTextAttnArgs& a, int unit, int gran) {
  TextUnit u = text_unit(a, unit, gran);
  if (u.rows > 0) u.block = (u.rows + gran - 1) / gran - 1 - u.block;
  return u;
}
// how many units there may be
inline long long text_units(const MdbTextAttnArgs& a, int gran) { return a.Sq / gran + static_cast<long long>(a.B); }
constexpr int TXT_FEW_SEQUENCES = 32;
// Packed and with gradients: whether the rows of a sequence have few keys. The rounding of their probabilities and of ds shows most in the result: P near 1/2 is off by up to
// 2^-8 of itself where the result's own rounding is off by 2^-9.3 on average, and ds = p (dp - do . o) is a difference of nearly equal terms. They go into their
// products as two bf16 terms. The sequence alone decides, so that a result's rounding does not depend on what else is packed. Relative errors of dq against 64 bits with one term / with two:
// sequences of two or three tokens 0.0026 to 0.0030 / 0.0017, of 200 0.0024 / 0.0017, of 1500 0.0024 / 0.0017, where two would take a training step of nine sequences of 20 to 1531
// (32 / 8 heads of 128) from 413 us to 484; 40 sequences of 128 223 us with two terms, 205 with one; 1500 and 1000 with a window of 200 186 and 168.
constexpr int TXT_FEW_ROWS = 256, TXT_SHORT_WINDOW = 128;
__device__ __forceinline__ bool text_is_fine(const MdbTextAttnArgs& a, int rows) { return rows <= TXT_FEW_ROWS || a.window <= TXT_SHORT_WINDOW; }
int text_make_units(const MdbTextAttnArgs& a, int gran, cudaStream_t st);

// rows before the first sequence and behind the last one, in turn; by whole warps. Where ends fall there are no units, so a CTA that had one need not look: then all rows, and a report.
template <typename F> __device__ __forceinline__ void text_rows_of_none(const MdbTextAttnArgs& a, bool look, int from, int step, F f) {
  int first = text_row_within(a, 0), last = text_row_within(a, a.B);
  if (look) {
    const int lane = threadIdx.x & 31;
    const bool fell = a.units != nullptr ? a.units[0].w < 0 : lane < a.B && text_row_within(a, lane + 1) < text_row_within(a, lane);
    if (__any_sync(0xffffffffu, fell)) {
      if (lane == 0) report_status(a.status, STATUS_BOUNDS, 187, a.B);
      first = last = 0;
    }
  }
  const int n = first + a.Sq - last;
  for (int i = from; i < n; i += step) f(i < first ? i : i - first + last);
}

__device__ __forceinline__ bool mbar_test_wait(uint64_t* bar, uint32_t parity) {
  uint32_t ok;
  asm volatile(
      "{\n"
      ".reg .pred P;\n"
      "mbarrier.test_wait.parity.shared::cta.b64 P, [%1], %2;\n"
      "selp.u32 %0, 1, 0, P;\n"
      "}\n"
      : "=r"(ok)
      : "r"(smem_u32(bar)), "r"(parity)
      : "memory");
  return ok != 0;
}

// maxima that keep NaN: a score that is not a number makes the row's reference NaN, and with it the whole row, as in a plain softmax
__device__ __forceinline__ float max_nan(float a, float b) {
  float d;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(d) : "f"(a), "f"(b));
  return d;
}
__device__ __forceinline__ float max3_nan(float a, float b, float c) {
  float d;
  asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
}

// mbar_wait in fewer instructions, by a whole warp: these kernels wait at many places, and what they do in between must stay in the instruction cache.
// PROBE: a look without the option to suspend comes first, which is shorter where the phase is over already; the issuing warp waits twice for each tile
// (8192 tokens, heads of 128, window 1024: 164 us, 171 without; training on 2 x 2048 tokens 280 us, 286). It is ten instructions more at each
// place: heads of 64, whose two CTAs per SM fill each other's gaps, lose by them (a prompt of 300 tokens 11.7 us, 11.0 without).
template <bool PROBE>
__device__ __forceinline__ bool text_wait(uint64_t* bar, uint32_t parity, volatile int* abort_flag) {
  if (PROBE && __all_sync(0xffffffffu, mbar_test_wait(bar, parity))) return true;
  uint64_t since = 0;
  uint32_t spins = 0;
  bool ok = true;
#pragma unroll 1
  while (!mbar_try_wait(bar, parity)) {
    if ((++spins & 63u) != 0) continue;
    const uint64_t now = globaltimer_ns();
    if (since == 0) since = now;
    if (now - since > MDB_WAIT_LIMIT_NS || *abort_flag) {
      *abort_flag = 1;
      ok = false;
      break;
    }
  }
  return __all_sync(0xffffffffu, ok);
}

// distributed shared memory of the cluster
__device__ __forceinline__ uint32_t ld_cluster_u32(uint32_t addr) {
  uint32_t v;
  asm volatile("ld.shared::cluster.u32 %0, [%1];" : "=r"(v) : "r"(addr) : "memory");
  return v;
}
__device__ __forceinline__ float ld_cluster_f32(uint32_t addr) { return __uint_as_float(ld_cluster_u32(addr)); }
__device__ __forceinline__ float4 ld_cluster_f32x4(uint32_t addr) {
  float4 v;
  asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(addr) : "memory");
  return v;
}

// bit i: i < n
__device__ __forceinline__ uint32_t bits_below(int n) { return n <= 0 ? 0u : n >= 32 ? 0xffffffffu : (1u << n) - 1u; }
// bit i: the query at position p sees key k0 + i
__device__ __forceinline__ uint32_t text_mask(const MdbTextAttnArgs& a, int valid, int p, int k0) {
  return bits_below(min(p + 1, valid) - k0) & (~bits_below(p - a.window + 1 - k0) | bits_below(a.sinks - k0));
}

// Distances from `near` on share one bucket per direction; text_bucket(rel) is constant beyond it on either side.
__host__ __device__ __forceinline__ int text_near(const MdbTextAttnArgs& a) { return a.n_borders > 0 ? a.borders[a.n_borders - 1] : a.exact; }
__device__ __forceinline__ int text_bucket(const MdbTextAttnArgs& a, int rel) {
  const int n = rel < 0 ? -rel : rel;
  int c = n;
  if (n >= a.exact) {
    c = a.exact;
    for (int i = 0; i < a.n_borders; ++i) c += n >= a.borders[i];
  }
  return c + (rel > 0 ? a.buckets / 2 : 0);
}

// The bias of one head by distance, for the distances -near - 254 .. near + 254 (all that a tile near the diagonal meets), in shared memory. Four
// copies, shifted by an element each: a thread reads four neighbours with one aligned 16-byte load, whatever its row; the distance between the
// copies lets 8 lanes of consecutive rows hit all banks.
struct TextLut {
  static __host__ __device__ __forceinline__ int entries(int near) { return 2 * near + 509; }
  static __host__ __device__ __forceinline__ int copy_floats(int near) { return (entries(near) + 3 + 31) / 32 * 32 + 8; }
  static __host__ __device__ __forceinline__ int bytes(int near) { return 4 * copy_floats(near) * 4; }

  float* copies;
  int near, ld;
  __device__ __forceinline__ TextLut(void* smem, int near_) : copies(static_cast<float*>(smem)), near(near_), ld(copy_floats(near_)) {}
  // By `warps` whole warps; the caller synchronises. Every warp takes some of the buckets, in the order of their distances, with one load for their
  // values, and stores each over its distances.
  __device__ __forceinline__ void set(const MdbTextAttnArgs& a, int head, int warp, int warps) const {
    const int mid = a.exact + a.n_borders, n = entries(near), lane = threadIdx.x & 31;
    const auto reach = [&](int c) { return c <= a.exact ? c : a.borders[c - a.exact - 1]; };      // first distance of a bucket of either direction
    const auto start = [&](int r) { return r <= 0 ? -near - 254 : r <= mid ? 1 - reach(mid - r + 1) : reach(r - mid); };
    const int mine = warp + lane * warps;
    float v = 0.f;
    if (mine <= 2 * mid) v = TXT_LOG2E * text_param(a.table, a.param_f32, static_cast<long long>(mine <= mid ? mid - mine : mine - mid + a.buckets / 2) * a.H + head);
    for (int k = 0, r = warp; r <= 2 * mid; ++k, r += warps) {
      const float u = __shfl_sync(0xffffffffu, v, k);
      const int lo = start(r) + near + 254, hi = r == 2 * mid ? n : start(r + 1) + near + 254;
      for (int i = lo + lane; i < hi; i += 32)
#pragma unroll
        for (int j = 0; j < 4; ++j) copies[j * ld + i + j] = u;
    }
  }
  __device__ __forceinline__ float before() const { return copies[0]; }                       // key far before the query, and behind it
  __device__ __forceinline__ float behind() const { return copies[entries(near) - 1]; }
  // where the biases of the distances d, d + 1, ... lie: 16-byte loads at multiples of four
  __device__ __forceinline__ const float* from(int d) const {
    const int i = near + 254 + d, j = -i & 3;
    return copies + j * ld + i + j;
  }
};

// lets `kern` have up to `bytes` of dynamic shared memory on the current device; once for each
constexpr int TXT_DEVICES = 64;
template <typename K>
inline int allow_smem(K kern, int bytes, bool (&ready)[TXT_DEVICES]) {
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e == cudaSuccess && dev < TXT_DEVICES && ready[dev]) return 0;
  if (e == cudaSuccess) e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
  if (e != cudaSuccess) return static_cast<int>(e);
  if (dev < TXT_DEVICES) ready[dev] = true;
  return 0;
}

// and clusters of up to 16 CTAs
template <typename K>
inline int allow_wide_clusters(K kern, bool (&ready)[TXT_DEVICES]) {
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e == cudaSuccess && dev < TXT_DEVICES && ready[dev]) return 0;
  if (e == cudaSuccess) e = cudaFuncSetAttribute(kern, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
  if (e != cudaSuccess) return static_cast<int>(e);
  if (dev < TXT_DEVICES) ready[dev] = true;
  return 0;
}

int text_attention_prompt(const MdbTextAttnArgs& a, cudaStream_t st);
bool text_attention_is_step(const MdbTextAttnArgs& a);
int text_attention_step(const MdbTextAttnArgs& a, cudaStream_t st);
long long text_attention_backward_floats(const MdbTextAttnArgs& a);
int text_attention_backward(const MdbTextAttnArgs& a, cudaStream_t st);

}  // namespace mdb
