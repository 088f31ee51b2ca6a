// Entry points of the language models' attention: causal grouped-query attention with a sliding window, a few first keys that stay visible and a
// learned sink logit per head, and attention over a whole prompt with a learned bias for buckets of relative positions.
//
//   s_ij = scale q_i . k_j (+ table[bucket(j - i), h]);  p_ij = exp(s_ij - lse_i) over the keys that i sees;  o_i = sum_j p_ij v_j
//   delta_i = do_i . o_i;  ds_ij = p_ij (do_i . v_j - delta_i)
//   dq_i = scale sum_j ds_ij k_j;  dk_j = scale sum_i ds_ij q_i;  dv_j = sum_i p_ij do_i   (the last two over the heads of a group)
//   dtable[b, h] = sum of ds_ij over the pairs of the bucket;  dsink[h] = -sum_i exp(sink_h - lse_i) delta_i
#include "text_attention.cuh"

namespace mdb {

static int check_args(const MdbTextAttnArgs* a) {
  if (a->B <= 0 || a->H <= 0 || a->Hkv <= 0 || a->H % a->Hkv != 0 || a->Sq <= 0 || a->Skv <= 0) return -1;
  if (a->Dh != 64 && a->Dh != 128) return -2;
  if (a->cu != nullptr && (a->Sq != a->Skv || a->sinks != 0 || a->table != nullptr || a->kv_len != nullptr || a->q_start_ptr != nullptr || a->q_start != 0)) return -7;
  if (a->window < 1 || a->window > TXT_FAR || a->sinks < 0 || !(a->scale > 0.f)) return -5;
  if (a->table == nullptr) return 0;
  if (a->Hkv != a->H || a->buckets < 4 || a->buckets > MDB_TEXT_MAX_BUCKETS * 64 / a->Dh || a->buckets % 2 != 0 || a->exact < 1 || a->n_borders < 0 ||
      a->exact + a->n_borders > a->buckets / 2 - 1 || a->n_borders > MDB_TEXT_MAX_BUCKETS / 2)
    return -6;
  int last = a->exact;
  for (int i = 0; i < a->n_borders; ++i) {
    if (a->borders[i] < last) return -6;
    last = a->borders[i];
  }
  return last > (a->Dh == 64 ? MDB_TEXT_MAX_NEAR_64 : MDB_TEXT_MAX_NEAR_128) ? -6 : 0;
}

// The units of more than 32 sequences, one block of threads: sequence after sequence, the last rows of each first
constexpr int TU_THREADS = 1024;
__global__ void __launch_bounds__(TU_THREADS) text_units_kernel(const __grid_constant__ MdbTextAttnArgs a, const int gran, const int units) {
  __shared__ int sums[TU_THREADS / 32], at[TU_THREADS];
  __shared__ int2 rows_of[TU_THREADS];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  bool falls = false;
  int before = 0;
  for (int b0 = 0; b0 < a.B; b0 += TU_THREADS) {
    const int b = b0 + threadIdx.x, first = b < a.B ? text_row_within(a, b) : 0, rows = b < a.B ? text_row_within(a, b + 1) - first : 0, n = max(rows + gran - 1, 0) / gran;
    falls = falls || rows < 0;
    int upto = n;
#pragma unroll
    for (int m = 1; m < 32; m <<= 1) {
      const int other = __shfl_up_sync(0xffffffffu, upto, m);
      if (lane >= m) upto += other;
    }
    __syncthreads();
    if (lane == 31) sums[warp] = upto;
    __syncthreads();
    int off = before, all = 0;
    for (int w = 0; w < TU_THREADS / 32; ++w) {
      off += w < warp ? sums[w] : 0;
      all += sums[w];
    }
    at[threadIdx.x] = off + upto - n;
    rows_of[threadIdx.x] = make_int2(first, rows);
    __syncthreads();
    for (int i = warp; i < TU_THREADS && b0 + i < a.B; i += TU_THREADS / 32) {
      const int blocks = (rows_of[i].y + gran - 1) / gran;
      for (int k = lane; k < blocks && static_cast<unsigned>(at[i] + k) < static_cast<unsigned>(units); k += 32) a.units[at[i] + k] = make_int4(rows_of[i].x, rows_of[i].y, blocks - 1 - k, b0 + i);
    }
    before += all;
  }
  const bool none = __syncthreads_or(falls);      // where ends fall there is no unit, and the first place says so
  for (int i = (none ? 0 : before) + threadIdx.x; i < units; i += TU_THREADS) a.units[i] = make_int4(0, 0, 0, none ? -1 : 0);
}
int text_make_units(const MdbTextAttnArgs& a, int gran, cudaStream_t st) {
  if (a.units == nullptr) return 0;
  text_units_kernel<<<1, TU_THREADS, 0, st>>>(a, gran, static_cast<int>(text_units(a, gran)));
  return static_cast<int>(cudaGetLastError());
}

}  // namespace mdb

extern "C" long long mdb_text_attention_units(const MdbTextAttnArgs* a) { return a->cu == nullptr || a->B <= mdb::TXT_FEW_SEQUENCES ? 0 : mdb::text_units(*a, 128); }
extern "C" int mdb_text_attention_fwd(const MdbTextAttnArgs* a, cudaStream_t st) {
  if (int r = mdb::check_args(a)) return r;
  return a->cu == nullptr && mdb::text_attention_is_step(*a) ? mdb::text_attention_step(*a, st) : mdb::text_attention_prompt(*a, st);
}

extern "C" long long mdb_text_attention_bwd_floats(const MdbTextAttnArgs* a) {
  return mdb::check_args(a) ? 0 : mdb::text_attention_backward_floats(*a);
}

extern "C" int mdb_text_attention_bwd(const MdbTextAttnArgs* a, cudaStream_t st) {
  if (int r = mdb::check_args(a)) return r;
  return mdb::text_attention_backward(*a, st);
}
