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

}  // namespace mdb

extern "C" int mdb_text_attention_fwd(const MdbTextAttnArgs* a, cudaStream_t st) {
  if (int r = mdb::check_args(a)) return r;
  return mdb::text_attention_is_step(*a) ? mdb::text_attention_step(*a, st) : mdb::text_attention_prompt(*a, st);
}

extern "C" long long mdb_text_attention_bwd_floats(const MdbTextAttnArgs* a) {
  return mdb::check_args(a) ? 0 : mdb::text_attention_backward_floats(*a);
}

extern "C" int mdb_text_attention_bwd(const MdbTextAttnArgs* a, cudaStream_t st) {
  if (int r = mdb::check_args(a)) return r;
  return mdb::text_attention_backward(*a, st);
}
