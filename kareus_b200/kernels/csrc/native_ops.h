// Entry points of libkareus_b200.so that the extension module of the 8-bit, Newton-Schulz and embedding calls uses
// (torch/opcalls.cpp).  The sources that define them include this too, so that a changed signature does not compile until both
// sides have it.
#pragma once
#include <cuda_runtime.h>

extern "C" {
int kb_fp8_quantize(const void* x, long rows, long cols, long ld, void* q, long ldq, void* s, void* qt, long ldqt, void* st,
                    int square, int fmt, cudaStream_t stream);
int kb_gemm_fp8(const void* A, const void* SA, int fmt_a, long lda, const void* B, const void* SB, int fmt_b, long ldb, void* C,
                long ldc, int M, int N, int K, int out_f32, int accumulate, int* status, cudaStream_t stream);
long kb_newton_schulz_bytes(long batch, long m, long n);
int kb_newton_schulz_launches(int batch, int m, int n, int steps);
int kb_newton_schulz(const void* x, int bf16, int batch, int m, int n, float a, float b, float c, int steps, float eps, float scale,
                     float scale_q, void* out, void* work, int* status, cudaStream_t stream);
int kb_embedding_fwd(const long* tokens, const void* w, void* out, long ntok, int H, long first, long rows, float scale,
                            cudaStream_t stream);
long kb_embedding_sorted_bytes(long ntok, int H);
int kb_embedding_sorted_launches(long ntok);
int kb_embedding_bwd_sorted(const long* tokens, const void* dout, float* grad, long ntok, int H, long first, long rows, float scale,
                            void* work, cudaStream_t stream);
}
