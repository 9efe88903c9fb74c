// Dense products with e4m3 weights: what oco_dense_* calls for OCO_FMT_F8_E4M3 (f8.cu).
#pragma once
#include "../../include/oco_moe.h"

namespace oco {

// A plan of one dense product; kind is OCO_DENSE_PROJECTION or OCO_DENSE_FFN_SILU_GATE. Errors as in the C ABI.
int f8_dense_create(const oco_dense_desc& desc, oco_moe_f8_plan** out);
int f8_dense_bind_codes(oco_moe_f8_plan* plan, const oco_dense_weights& w);
int f8_dense_bind_scales(oco_moe_f8_plan* plan, const oco_dense_scales& s);
int f8_dense_forward(oco_moe_f8_plan* plan, const uint16_t* x, uint16_t* y, int rows, void* cuda_stream);

}  // namespace oco
