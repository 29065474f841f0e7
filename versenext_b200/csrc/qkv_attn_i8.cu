#include "qkv_attn_tc.cuh"

int32_t qkv_attention_i8(vn_qkv* c, const QkvAttnArgs& a) { return qkv_detail::pick<QKV_I8>(c, a); }
