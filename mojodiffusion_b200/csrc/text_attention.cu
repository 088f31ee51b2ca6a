// Attention of the language models: causal grouped-query attention with a sliding window, a few first keys that stay visible and a learned
// sink logit per head (mask kind CAUSAL), and attention over a whole prompt with a learned bias for buckets of relative positions (BIAS).
//
//   s_ij = scale q_i . k_j (+ table[bucket(j - i), h]);  p_ij = exp(s_ij - lse_i) over the keys that i sees;  o_i = sum_j p_ij v_j
//   delta_i = do_i . o_i;  ds_ij = p_ij (do_i . v_j - delta_i)
//   dq_i = scale sum_j ds_ij k_j;  dk_j = scale sum_i ds_ij q_i;  dv_j = sum_i p_ij do_i   (the last two over the heads of a group)
//   dtable[b, h] = sum of ds_ij over the pairs of the bucket;  dsink[h] = -sum_i exp(sink_h - lse_i) delta_i
//
// This is the plain form on CUDA cores: one warp per row, all sums in fp32.
#include "text_attention.cuh"

#include <string.h>

namespace mdb {

template <int DH> struct Row {
  static constexpr int N = DH / 32;
  float x[N];
  __device__ __forceinline__ void load(const void* base, long long off, int lane) {
    const __nv_bfloat16* p = static_cast<const __nv_bfloat16*>(base) + off + lane * N;
#pragma unroll
    for (int i = 0; i < N; ++i) x[i] = __bfloat162float(p[i]);
  }
  __device__ __forceinline__ void store(void* base, long long off, int lane, float f) const {
    __nv_bfloat16* p = static_cast<__nv_bfloat16*>(base) + off + lane * N;
#pragma unroll
    for (int i = 0; i < N; ++i) p[i] = __float2bfloat16_rn(x[i] * f);
  }
  __device__ __forceinline__ float dot(const Row& o) const {
    float s = 0.f;
#pragma unroll
    for (int i = 0; i < N; ++i) s += x[i] * o.x[i];
#pragma unroll
    for (int m = 16; m > 0; m >>= 1) s += __shfl_xor_sync(0xffffffffu, s, m);
    return s;
  }
  __device__ __forceinline__ void zero() {
#pragma unroll
    for (int i = 0; i < N; ++i) x[i] = 0.f;
  }
  __device__ __forceinline__ void add(const Row& o, float f) {
#pragma unroll
    for (int i = 0; i < N; ++i) x[i] += f * o.x[i];
  }
  __device__ __forceinline__ void scale(float f) {
#pragma unroll
    for (int i = 0; i < N; ++i) x[i] *= f;
  }
};

__device__ __forceinline__ long long at(const long long* st, int b, int s, int h) {
  return b * st[0] + static_cast<long long>(s) * st[1] + h * st[2];
}

template <int DH>
__global__ void text_dq_kernel(const MdbTextAttnArgs a) {
  const long long w = (blockIdx.x * static_cast<long long>(blockDim.x) + threadIdx.x) >> 5;
  const int lane = threadIdx.x & 31;
  if (w >= static_cast<long long>(a.B) * a.H * a.Sq) return;
  const int i = static_cast<int>(w % a.Sq), h = static_cast<int>((w / a.Sq) % a.H), b = static_cast<int>(w / (static_cast<long long>(a.Sq) * a.H));
  const int g = h / (a.H / a.Hkv);
  const TextSight s = text_sight(a, b);
  const int p = s.start + i;
  const int hi = (a.table == nullptr) ? min(p + 1, s.valid) : s.valid;
  const int lo = (a.table == nullptr) ? max(p - a.window + 1, 0) : 0;
  Row<DH> q, o, d, dq;
  q.load(a.q, at(a.q_strides, b, i, h), lane);
  o.load(a.o, at(a.o_strides, b, i, h), lane);
  d.load(a.dout, at(a.do_strides, b, i, h), lane);
  const float delta = d.dot(o), lse = a.lse[w];
  if (lane == 0) a.delta[w] = delta;
  dq.zero();
  float* part = a.d_table != nullptr ? a.table_ws + w * a.buckets : nullptr;
  if (part != nullptr) {
    for (int c = lane; c < a.buckets; c += 32) part[c] = 0.f;
    __syncwarp();
  }
  for (int j = 0; j < hi; ++j) {
    if (j >= a.sinks && j < lo) j = lo;
    if (j >= hi) break;
    Row<DH> k, v;
    k.load(a.k, at(a.k_strides, b, j, g), lane);
    v.load(a.v, at(a.v_strides, b, j, g), lane);
    float x = q.dot(k) * a.scale;
    const int c = a.table != nullptr ? text_bucket(a, j - i) : 0;
    if (a.table != nullptr) x += text_param(a.table, a.param_f32, static_cast<long long>(c) * a.H + h);
    const float ds = exp2f(x * TXT_LOG2E - lse) * (d.dot(v) - delta);
    dq.add(k, ds);
    if (part != nullptr && lane == 0) part[c] += ds;
  }
  dq.store(a.dq, at(a.dq_strides, b, i, h), lane, a.scale);
}

template <int DH>
__global__ void text_dkv_kernel(const MdbTextAttnArgs a) {
  const long long w = (blockIdx.x * static_cast<long long>(blockDim.x) + threadIdx.x) >> 5;
  const int lane = threadIdx.x & 31;
  if (w >= static_cast<long long>(a.B) * a.Hkv * a.Skv) return;
  const int j = static_cast<int>(w % a.Skv), g = static_cast<int>((w / a.Skv) % a.Hkv), b = static_cast<int>(w / (static_cast<long long>(a.Skv) * a.Hkv));
  const TextSight s = text_sight(a, b);
  Row<DH> k, v, dk, dv;
  k.load(a.k, at(a.k_strides, b, j, g), lane);
  v.load(a.v, at(a.v_strides, b, j, g), lane);
  dk.zero();
  dv.zero();
  const int rep = a.H / a.Hkv;
  const int i0 = (a.table == nullptr) ? max(j - s.start, 0) : 0;
  const int i1 = j >= s.valid ? 0 : ((a.table == nullptr) && j >= a.sinks) ? static_cast<int>(min(static_cast<long long>(a.Sq), static_cast<long long>(j) + a.window - s.start)) : a.Sq;
  for (int h = g * rep; h < (g + 1) * rep; ++h)
    for (int i = i0; i < i1; ++i) {
      Row<DH> q, d;
      q.load(a.q, at(a.q_strides, b, i, h), lane);
      d.load(a.dout, at(a.do_strides, b, i, h), lane);
      const long long r = (static_cast<long long>(b) * a.H + h) * a.Sq + i;
      float x = q.dot(k) * a.scale;
      if (a.table != nullptr) x += text_param(a.table, a.param_f32, static_cast<long long>(text_bucket(a, j - i)) * a.H + h);
      const float e = exp2f(x * TXT_LOG2E - a.lse[r]);
      dv.add(d, e);
      dk.add(q, e * (d.dot(v) - a.delta[r]));
    }
  dk.store(a.dk, at(a.dk_strides, b, j, g), lane, a.scale);
  dv.store(a.dv, at(a.dv_strides, b, j, g), lane, 1.f);
}

// dsink of one head per block; the order of the sum is fixed by the launch shape
__global__ void text_dsink_kernel(const MdbTextAttnArgs a) {
  __shared__ float part[256];
  const int h = blockIdx.x;
  const float sink = text_param(a.sink_logits, a.param_f32, h);
  float s = 0.f;
  for (long long r = threadIdx.x; r < static_cast<long long>(a.B) * a.Sq; r += 256) {
    const long long at_ = ((r / a.Sq) * a.H + h) * a.Sq + r % a.Sq;
    s += exp2f(sink * TXT_LOG2E - a.lse[at_]) * a.delta[at_];
  }
  part[threadIdx.x] = s;
  __syncthreads();
  for (int n = 128; n > 0; n >>= 1) {
    if (threadIdx.x < n) part[threadIdx.x] += part[threadIdx.x + n];
    __syncthreads();
  }
  if (threadIdx.x == 0) {
    if (a.param_f32) static_cast<float*>(a.d_sink)[h] = -part[0];
    else static_cast<__nv_bfloat16*>(a.d_sink)[h] = __float2bfloat16_rn(-part[0]);
  }
}

// dtable[bucket, h]: one block each
__global__ void text_dtable_kernel(const MdbTextAttnArgs a) {
  __shared__ float part[256];
  const int h = blockIdx.x, c = blockIdx.y;
  float s = 0.f;
  for (long long r = threadIdx.x; r < static_cast<long long>(a.B) * a.Sq; r += 256)
    s += a.table_ws[(((r / a.Sq) * a.H + h) * a.Sq + r % a.Sq) * a.buckets + c];
  part[threadIdx.x] = s;
  __syncthreads();
  for (int n = 128; n > 0; n >>= 1) {
    if (threadIdx.x < n) part[threadIdx.x] += part[threadIdx.x + n];
    __syncthreads();
  }
  if (threadIdx.x == 0) {
    const long long to = static_cast<long long>(c) * a.H + h;
    if (a.param_f32) static_cast<float*>(a.d_table)[to] = part[0];
    else static_cast<__nv_bfloat16*>(a.d_table)[to] = __float2bfloat16_rn(part[0]);
  }
}

static int check_args(const MdbTextAttnArgs* a) {
  if (a->B <= 0 || a->H <= 0 || a->Hkv <= 0 || a->H % a->Hkv != 0 || a->Sq <= 0 || a->Skv <= 0) return -1;
  if (a->Dh != 64 && a->Dh != 128) return -2;
  if (a->window < 1 || a->window > TXT_FAR || a->sinks < 0 || !(a->scale > 0.f)) return -5;
  if (a->table != nullptr && (a->buckets < 4 || a->buckets > MDB_TEXT_MAX_BUCKETS || a->n_borders < 0 || a->n_borders > MDB_TEXT_MAX_BUCKETS / 4 ||
                              a->exact < 1 || a->exact + a->n_borders > a->buckets / 2 - 1 || (a->n_borders == 0 && a->exact > MDB_TEXT_MAX_DISTANCE) ||
                              (a->n_borders > 0 && a->borders[a->n_borders - 1] > MDB_TEXT_MAX_DISTANCE)))
    return -6;
  return 0;
}
static unsigned blocks_for(long long rows) { return static_cast<unsigned>((rows * 32 + 127) / 128); }

}  // namespace mdb

extern "C" int mdb_text_attention_fwd(const MdbTextAttnArgs* a, cudaStream_t st) {
  using namespace mdb;
  if (int r = check_args(a)) return r;
  return text_attention_prompt(*a, st);
}

extern "C" long long mdb_text_attention_bwd_floats(const MdbTextAttnArgs* a) {
  return static_cast<long long>(a->B) * a->H * a->Sq * a->buckets;
}

extern "C" int mdb_text_attention_bwd(const MdbTextAttnArgs* a, cudaStream_t st) {
  using namespace mdb;
  if (int r = check_args(a)) return r;
  const unsigned nq = blocks_for(static_cast<long long>(a->B) * a->H * a->Sq), nk = blocks_for(static_cast<long long>(a->B) * a->Hkv * a->Skv);
  if (a->Dh == 128) {
    text_dq_kernel<128><<<nq, 128, 0, st>>>(*a);
    text_dkv_kernel<128><<<nk, 128, 0, st>>>(*a);
  } else {
    text_dq_kernel<64><<<nq, 128, 0, st>>>(*a);
    text_dkv_kernel<64><<<nk, 128, 0, st>>>(*a);
  }
  if (a->d_sink != nullptr) text_dsink_kernel<<<a->H, 256, 0, st>>>(*a);
  if (a->d_table != nullptr) text_dtable_kernel<<<dim3(a->H, a->buckets), 256, 0, st>>>(*a);
  return static_cast<int>(cudaGetLastError());
}
