// SPDX-License-Identifier: Unlicense
//
// Internal interface of the 8-bit linear layers (linear_i8.cu, tc_i8.cu).

#pragma once

#include "opcheck.cuh"

namespace coreg {

// C = act((A B^T) sa sb + bias) + R as in ops_gemm_i8 (ops_b200.h); the rows
// of A and B start at multiples of 16 bytes.
struct I8Gemm {
    int M, N, K;
    const int8_t *A;
    long lda;
    const float *sa;
    const int8_t *B;
    long ldb;
    const float *sb;
    const float *bias; // per column or NULL
    void *C;
    long ldc;
    const void *R; // C's layout and type, or NULL
    int c_bf16;
    int act;
    float slope;
};

// On the tcgen05 integer tensor cores; false (nothing launched) where no
// tensor map describes the operands.
bool gemm_i8_tc(cudaStream_t st, const I8Gemm &g, int sms);

}  // namespace coreg
