// The entry points on 8-bit rows and score rows for callers that know which device owns the buffers (tensors.cpp): vdb_*_dev of vdbmi.h
// with that device in front, and without asking the runtime about each buffer; device < 0 asks.
#pragma once
#include "../../include/vdbmi.h"

extern "C" {
vdb_status vdb_q8_quantize_on(int device, const void* d_rows, vdb_dtype dtype, size_t stride, const vdb_q8_rows* out, void* stream);
vdb_status vdb_q8_score_on(int device, const vdb_q8_rows* queries, const vdb_q8_rows* base, vdb_metric metric, float* d_out, size_t out_stride, void* stream);
vdb_status vdb_score_adjust_on(int device, const float* d_scores, size_t stride, size_t nq, size_t n, vdb_metric metric, const vdb_score_adjust* how,
                               float* d_out, size_t out_stride, void* stream);
}
