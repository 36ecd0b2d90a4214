// cb_gemm_i8.hip — matrix product in 8-bit integers with a scale per token and per channel:
//   C[m][n] = sa[m] sb[n] sum_k A[m][k] B[n][k]  + bias[n] + R[m][n]
// The sum is exact in 32-bit integers (128^2 K < 2^31), so no order of summation changes it.
//
// Tile kernel: BM x BN outputs a block of 4 waves (2 x 2), k-tiles of 128 (one 128-byte row a tile row) by LDS-DMA into a ring of two stages;
// piece c of row r lies at place c ^ ((r >> 1) & 7), as in cb_gemm_glds.hip. v_mfma_i32_32x32x32_i8: a lane holds 16 bytes of a row.
#include "cb_device.h"
#include "cb_i8.h"
#include <type_traits>

namespace cb {

typedef int i32x4 __attribute__((ext_vector_type(4)));
typedef int i32x16 __attribute__((ext_vector_type(16)));
typedef __attribute__((address_space(3))) void* lds_vp;
constexpr int I8_OOB = -16;

__device__ __forceinline__ __amdgpu_buffer_rsrc_t i8_srd(const void* p) {
    return __builtin_amdgcn_make_buffer_rsrc(const_cast<void*>(p), 0, 0x7FFFFFFF, 0x00020000);
}
__device__ __forceinline__ int i8_xcd(int id, int n) {
    const int per = n >> 3, rem = n & 7, x = id & 7, y = id >> 3;
    return x * per + min(x, rem) + y;
}
// one output: scales, bias, residual, one rounding
template <typename T> __device__ __forceinline__ float i8_finish(const GemmI8Args& a, int acc, float sa, int m, int n) {
    float v = (float)acc * (sa * a.sb[n]);
    if (a.bias) v += a.bias[n];
    if (a.R) v += ld1(static_cast<const T*>(a.R) + (long)m * a.ldr + n);
    return v;
}

template <typename T, int BM, int BN>
__global__ __launch_bounds__(256) void gemm_i8_kernel(const GemmI8Args a, const int tm, const int tn) {
#ifdef __HIP_DEVICE_COMPILE__      // the host pass needs the launch stub alone
    constexpr int RB = 128, AT = BM * RB, BT = BN * RB, STAGE = AT + BT, NA = AT / 4096, NB = BT / 4096, WM = BM / 64, WN = BN / 64;
    extern __shared__ __attribute__((aligned(16))) char lds_i8[];
    const int tid = threadIdx.x, lane = tid & 63, ml = lane & 31, kl = lane >> 5;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6), wr = wave >> 1, wc = wave & 1;
    const int item = i8_xcd(blockIdx.x, gridDim.x);
    const int m0 = item / tn * BM, n0 = (item - item / tn * tn) * BN;
    const __amdgpu_buffer_rsrc_t srdA = i8_srd(a.A + (long)m0 * a.lda), srdB = i8_srd(a.B + (long)n0 * a.ldb);
    int ao[NA], bo[NB], kc[NA > NB ? NA : NB];
#pragma unroll
    for (int i = 0; i < (NA > NB ? NA : NB); ++i) {
        const int idx = tid + 256 * i, r = idx >> 3, c = ((idx & 7) ^ ((r >> 1) & 7)) * 16;
        kc[i] = c;
        if (i < NA) ao[i] = m0 + r < a.M ? (int)((long)r * a.lda + c) : I8_OOB;
        if (i < NB) bo[i] = n0 + r < a.N ? (int)((long)r * a.ldb + c) : I8_OOB;
    }
    const int nk = (a.K + RB - 1) / RB, wbase = wave * 1024;
    auto stage = [&](int t) {
        char* d = lds_i8 + (t & 1) * STAGE + wbase;
        const int k0 = t * RB;
#pragma unroll
        for (int i = 0; i < NA; ++i)
            __builtin_amdgcn_raw_ptr_buffer_load_lds(srdA, (lds_vp)(d + i * 4096), 16, k0 + kc[i] < a.K && ao[i] >= 0 ? ao[i] + k0 : I8_OOB, 0, 0, 0);
#pragma unroll
        for (int i = 0; i < NB; ++i)
            __builtin_amdgcn_raw_ptr_buffer_load_lds(srdB, (lds_vp)(d + AT + i * 4096), 16, k0 + kc[i] < a.K && bo[i] >= 0 ? bo[i] + k0 : I8_OOB, 0, 0, 0);
    };
    i32x16 acc[WM][WN];
#pragma unroll
    for (int i = 0; i < WM; ++i)
#pragma unroll
        for (int j = 0; j < WN; ++j)
#pragma unroll
            for (int r = 0; r < 16; ++r) acc[i][j][r] = 0;
    const int sw = (ml >> 1) & 7;
    const int aoff = (wr * (BM / 2) + ml) * RB, boff = AT + (wc * (BN / 2) + ml) * RB;
    stage(0);
    for (int t = 0; t < nk; ++t) {
        asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
        __builtin_amdgcn_s_barrier();
        asm volatile("" ::: "memory");
        if (t + 1 < nk) stage(t + 1);
        const char* S = lds_i8 + (t & 1) * STAGE;
#pragma unroll
        for (int s = 0; s < 4; ++s) {                            // 32 k a step: lane (kl, ml) holds pieces 2s + kl
            const int co = ((2 * s + kl) ^ sw) * 16;
            i32x4 av[WM], bv[WN];
#pragma unroll
            for (int i = 0; i < WM; ++i) av[i] = *reinterpret_cast<const i32x4*>(S + aoff + i * 32 * RB + co);
#pragma unroll
            for (int j = 0; j < WN; ++j) bv[j] = *reinterpret_cast<const i32x4*>(S + boff + j * 32 * RB + co);
#pragma unroll
            for (int i = 0; i < WM; ++i)
#pragma unroll
                for (int j = 0; j < WN; ++j) acc[i][j] = __builtin_amdgcn_mfma_i32_32x32x32_i8(av[i], bv[j], acc[i][j], 0, 0, 0);
        }
    }
#pragma unroll
    for (int i = 0; i < WM; ++i)
#pragma unroll
        for (int r = 0; r < 16; ++r) {
            const int m = m0 + wr * (BM / 2) + i * 32 + (r & 3) + 8 * (r >> 2) + 4 * kl;
            if (m >= a.M) continue;
            const float sa = a.sa[m];
#pragma unroll
            for (int j = 0; j < WN; ++j) {
                const int n = n0 + wc * (BN / 2) + j * 32 + ml;
                if (n < a.N) st1(static_cast<T*>(a.C) + (long)m * a.ldc + n, i8_finish<T>(a, acc[i][j][r], sa, m, n));
            }
        }
#endif
}

// ---------------------------------------------------------------- host side
size_t gemm_i8_ws_bytes(const GemmI8Args& a) { return 0; }
template <typename T, int BM, int BN> static void i8_go(const Launch& L, const GemmI8Args& a) {
    const int tm = (int)cdiv(a.M, BM), tn = (int)cdiv(a.N, BN);
    L.count();
    if (L.stats) { L.stats->gemm_flops += 2.0 * a.M * a.N * (double)a.K; L.stats->gemm_launches++; }
    if (L.dry) return;
    constexpr int lds = 2 * (BM + BN) * 128;
    set_dyn_lds(reinterpret_cast<const void*>(&gemm_i8_kernel<T, BM, BN>), 160 * 1024);
    hipLaunchKernelGGL((gemm_i8_kernel<T, BM, BN>), dim3((unsigned)tm * tn), dim3(256), lds, L.stream, a, tm, tn);
    CB_HIP(hipGetLastError());
}
void gemm_i8(const Launch& L, const GemmI8Args& a, void* ws) {
    CB_DT_SWITCH(a.dt, T, i8_go<T, 64, 64>(L, a));
}

}  // namespace cb
