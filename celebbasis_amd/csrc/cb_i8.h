// cb_i8.h — arguments of the residual RMS norm, of rows brought to 8 bits (cb_norm_i8.hip) and of the 8-bit product (cb_gemm_i8.hip)
#pragma once
#include "cb_common.h"

namespace cb {

struct RmsArgs {
    DType dt = DT_F32;
    long rows = 0; int C = 0; float eps = 0.f;
    const void* x = nullptr; long ldx = 0;
    const void* r = nullptr; long ldr = 0;           // residual (may be absent)
    const float* gamma = nullptr;
    void* h = nullptr; long ldh = 0;                 // held sum x + r (may be absent: forward without it)
    void* y = nullptr; long ldy = 0;                 // normed output in dt, or
    int8_t* q = nullptr; long ldq = 0; float* scale = nullptr;   // ... in 8 bits with a scale per row
    float* rstd = nullptr;
    // backward
    const void* dy = nullptr; long lddy = 0;
    const void* dres = nullptr; long lddres = 0;
    void* dh = nullptr; long lddh = 0;
    float* dgamma = nullptr; float* part = nullptr;
};
void k_rmsnorm_fwd(const Launch& L, const RmsArgs& a);
size_t rmsnorm_bwd_ws_bytes(long rows, int C);
void k_rmsnorm_bwd(const Launch& L, const RmsArgs& a);
// rows of x to 8 bits: scale = max|x| / 127, q = rint(x * 127 / max|x|); columns C .. ceil16(C) of q are zeroed
void k_quantize_rows(const Launch& L, const RmsArgs& a);

struct GemmI8Args {
    const int8_t* A = nullptr; const int8_t* B = nullptr;   // [M][lda], [N][ldb]: K contiguous
    int M = 0, N = 0, K = 0;
    long lda = 0, ldb = 0, ldc = 0, ldr = 0;
    const float* sa = nullptr; const float* sb = nullptr; const float* bias = nullptr;
    const void* R = nullptr; void* C = nullptr;
    DType dt = DT_F32;                                       // of C and R
    int* part = nullptr; int nsplit = 1;                     // [nsplit][M][N] sums of a split K axis
};
size_t gemm_i8_ws_bytes(const GemmI8Args& a);
void gemm_i8(const Launch& L, const GemmI8Args& a, void* ws);

constexpr int RMS_MAX_C = 16384, I8_MAX_K = 131071 / 16 * 16;    // 128 * 128 * K stays below 2^31

}  // namespace cb
