// Matrix-product problem description shared by the tensor-core and CUDA-core
// kernels.  Strides are in elements; `c` has unit column stride.
#pragma once

#include <cuda_runtime.h>

#include <cstdint>

namespace tpb {

struct GemmProblem {
    int dtype;
    int64_t M, N, K, batch;
    const void* a;  // A[b][m][k] at a + b*sa_b + m*sa_m + k*sa_k
    int64_t sa_b, sa_m, sa_k;
    const void* b;  // B[b][k][n] at b + b*sb_b + k*sb_k + n*sb_n
    int64_t sb_b, sb_k, sb_n;
    void* c;        // C[b][m][n] at c + b*sc_b + m*sc_m + n
    int64_t sc_b, sc_m;
    const void* cin;  // optional addend, any strides (0 = broadcast)
    int64_t sci_b, sci_m, sci_n;
    double alpha, beta;
    int flags;
    // Fused epilogue (tp_b200_gemm_epilogue): 0 none, 1 gelu (aux receives
    // the pre-activation), 2 gelu_backward (aux holds the activation's
    // input).  aux: [M x N], unit column stride, row stride saux_m.
    int epi;
    void* aux;
    int64_t saux_m;
};

void gemm_simt(const GemmProblem& p, int dev, cudaStream_t stream);
// False when the problem does not fit the tensor-core kernel's constraints
// (dtype, TMA alignment); nothing has been launched then.
bool gemm_tc(const GemmProblem& p, int dev, cudaStream_t stream);

// A feed-forward product (tp_b200_layer_forward and the products of
// tp_b200_layer_backward): y = epilogue(x w^T), x [M, K] and w [parts * N, K];
// parts 2: gate rows, then up rows.
struct FfnProblem {
    int dtype;
    int64_t M, N, K;
    int parts;
    const void* x;         // element (m, k) at x + m * sx_m + k * sx_k
    int64_t sx_m, sx_k;
    const void* w;         // element (n, k) at w + n * sw_n + k * sw_k
    int64_t sw_n, sw_k;
    void* y;               // [M, N], unit column stride
    int64_t sy_m;
    const void* bias;      // [parts * N] or null
    const void* residual;  // [M, N] or null
    int64_t sres_m;
    void* saved;           // [M, parts, N] contiguous or null
    int8_t* values;        // the same in 8 bits, or null
    uint8_t* exponents;
    int act;
    int flags;
};

// 16-bit floats: sx_k and sw_k 1; or, without an epilogue, sw_n 1 (dz w), or
// sx_m and sw_n 1 (dz^T x).  False when x
// or w does not fit the tensor maps (rows off 16-byte boundaries) or K is 0;
// nothing has been launched then.
bool gemm_ffn(const FfnProblem& q, int dev, cudaStream_t stream);
// The same for few rows; x and w fit the tensor maps.
void gemm_few(const FfnProblem& q, int dev, cudaStream_t stream);
double gemm_few_us(const FfnProblem& q, int dev);  // its estimated time
// float32: sx_k and sw_k 1, or sw_n 1, or sx_m and sw_n 1; K >= 1.
void gemm_f32(const FfnProblem& q, int dev, cudaStream_t stream);

}  // namespace tpb
