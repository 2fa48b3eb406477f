// q8.h — the 8-bit row operators behind jhq_q8_* of include/jhq.h: argument
// checks and launches, asynchronous on the stream, on the current device.
#pragma once
#include <cuda_runtime.h>

#include "jhq_common.h"

namespace jhq {

// Checks shared by the operators; each throws JHQ_EINVAL with `what` in front.
void q8_check_view(const jhq_view* v, const char* what);
void q8_check_rows(const jhq_q8_rows* r, const char* what);

void q8_rms_norm(const jhq_view* x, const jhq_view* residual, const jhq_view* weight, float eps,
                 const jhq_view* residual_out, const jhq_q8_rows* out, cudaStream_t s);
void q8_matmul(const jhq_q8_rows* x, const jhq_q8_rows* w, const jhq_view* bias, const jhq_view* out,
               cudaStream_t s);
void q8_write(const jhq_view* x, const int64_t* slots, const jhq_q8_rows* cache, cudaStream_t s);
void q8_read(const jhq_q8_rows* cache, const int64_t* slots, const jhq_view* out, cudaStream_t s);

// Whether a bounded device wait on the current device gave up; clears the mark.
bool q8_take_error();

}  // namespace jhq
