#include "qkv_attn_tc.cuh"

int32_t qkv_attention_e4m3(vn_qkv* c, const QkvAttnArgs& a) { return qkv_detail::pick<QKV_E4M3>(c, a); }
