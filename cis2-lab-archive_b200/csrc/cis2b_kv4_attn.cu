// cis2b_kv4_attn.cu -- causal attention over the 4-bit key/value cache
// (include/cis2b.h, cis2b_kv4_attention).
#include "cis2b_kv4_attn.cuh"

using namespace cis2b;

extern "C" int cis2b_kv4_workspace(const cis2b_kv4_cache *c, const cis2b_kv4_attn *a, uint64_t *out_bytes) {
  if (int rc = kv4_check_cache(c, false)) return rc;
  if (int rc = check_attn(c, a)) return rc;
  if (!out_bytes) return kv4_fail(CIS2B_ERR_ARG, "out_bytes is NULL");
  *out_bytes = shape_of(c, a).bytes;
  return CIS2B_OK;
}

extern "C" int cis2b_kv4_attention(const cis2b_kv4_cache *c, const cis2b_kv4_attn *a, void *stream) {
  return run_attention<Rows::CAUSAL>(c, a, AttArgs{}, stream);
}
