// cb_gemm_i8.hip — matrix product in 8-bit integers with a scale per token and per channel:
//   C[m][n] = sa[m] sb[n] sum_k A[m][k] B[n][k]  + bias[n] + R[m][n]
// The sum is exact in 32-bit integers (128^2 K < 2^31), so no order of summation changes it.
//
// A row of 128 k is 128 bytes, as a row of 64 k is in bf16, and a lane of v_mfma_i32_32x32x32_i8 holds 16 bytes of a row: the LDS images, their
// swizzle (piece c of row r at place c ^ ((r >> 1) & 7)) and the schedules of cb_gemm_glds.hip and cb_gemm_bf16_p8.hip hold byte for byte.
// Three kernels:
//   gemm_i8_few    up to 64 tokens: bound by reading the weights once. No LDS ring: 8 waves split K, each streams its part of 16 or 32 weight rows
//                  into registers and multiplies it with the tokens (from L2) in v_mfma_i32_16x16x64_i8; the waves' sums meet in LDS.
//   gemm_i8        64 x 64 or 128 x 128 outputs a block of 4 waves, LDS-DMA ring of two stages. Few tiles: K is split over blocks, 32-bit sums go to
//                  the workspace and one more kernel adds them (exact: any order gives the same).
//   gemm_i8_p8     256 x 256 outputs a block of 8 waves in the four-phase schedule that cb_gemm_bf16_p8.hip explains.
#include "cb_device.h"
#include "cb_i8.h"
#include <algorithm>
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
template <typename T> __device__ __forceinline__ void i8_put(const GemmI8Args& a, int acc, int m, int n) {
    float v = (float)acc * (a.sa[m] * a.sb[n]);
    if (a.bias) v += a.bias[n];
    if (a.R) v += ld1(static_cast<const T*>(a.R) + (long)m * a.ldr + n);
    st1(static_cast<T*>(a.C) + (long)m * a.ldc + n, v);
}
template <typename T> __device__ __forceinline__ void i8_ld8(const T* p, float (&v)[8]) {
    const float4 x = ld4(p), y = ld4(p + 4);
    v[0] = x.x; v[1] = x.y; v[2] = x.z; v[3] = x.w; v[4] = y.x; v[5] = y.y; v[6] = y.z; v[7] = y.w;
}
template <typename T> __device__ __forceinline__ void i8_st8(T* p, const float (&v)[8]) {
    if constexpr (sizeof(T) == 2) {
        bf16x8_t o;
#pragma unroll
        for (int e = 0; e < 8; ++e) o[e] = (bf16_t)v[e];
        *reinterpret_cast<bf16x8_t*>(p) = o;
    } else { st4(p, make_float4(v[0], v[1], v[2], v[3])); st4(p + 4, make_float4(v[4], v[5], v[6], v[7])); }
}
// 8 consecutive outputs of a row; `vec`: they are inside N and C, R may be accessed in 16-byte pieces
template <typename T> __device__ __forceinline__ void i8_put8(const GemmI8Args& a, const int (&acc)[8], const float (&sb)[8], const float (&bias)[8], int m, int n, bool vec) {
    if (!vec) {
        for (int e = 0; e < 8; ++e) if (n + e < a.N) i8_put<T>(a, acc[e], m, n + e);
        return;
    }
    const float sa = a.sa[m];
    float v[8], r[8];
    if (a.R) i8_ld8(static_cast<const T*>(a.R) + (long)m * a.ldr + n, r);
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        v[e] = (float)acc[e] * (sa * sb[e]);
        if (a.bias) v[e] += bias[e];
        if (a.R) v[e] += r[e];
    }
    i8_st8(static_cast<T*>(a.C) + (long)m * a.ldc + n, v);
}
// a wave's ROWS x COLS sums, parked in its own LDS (S), to the outputs at (m0, n0): a lane takes 8 consecutive columns of a row
template <typename T, int ROWS, int COLS>
__device__ __forceinline__ void i8_finish(const GemmI8Args& a, const int* S, int m0, int n0, int lane, bool al, int* part) {
    constexpr int LPR = COLS / 8, RPP = 64 / LPR;
    const int rs = lane / LPR, cc = (lane % LPR) * 8, n = n0 + cc;
    if (n >= a.N) return;
    const bool vec = al && n + 8 <= a.N;
    float sb[8], bias[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) { sb[e] = n + e < a.N ? a.sb[n + e] : 0.f; bias[e] = a.bias && n + e < a.N ? a.bias[n + e] : 0.f; }
#pragma unroll
    for (int p = 0; p < ROWS / RPP; ++p) {
        const int r = p * RPP + rs, m = m0 + r;
        if (m >= a.M) continue;
        const i32x4 x = *reinterpret_cast<const i32x4*>(S + r * COLS + cc), y = *reinterpret_cast<const i32x4*>(S + r * COLS + cc + 4);
        const int v[8] = {x[0], x[1], x[2], x[3], y[0], y[1], y[2], y[3]};
        if (part) {
            for (int e = 0; e < 8; ++e) if (n + e < a.N) part[(long)m * a.N + n + e] = v[e];
        } else i8_put8<T>(a, v, sb, bias, m, n, vec);
    }
}
// outputs and residual can be accessed in 16-byte pieces
template <typename T> __device__ __forceinline__ bool i8_aligned(const GemmI8Args& a) {
    const long e = 16 / sizeof(T);
    return ((reinterpret_cast<uintptr_t>(a.C) & 15) == 0) && a.ldc % e == 0 && (!a.R || (((reinterpret_cast<uintptr_t>(a.R) & 15) == 0) && a.ldr % e == 0));
}
// block -> tile: a contiguous run of tiles for each XCD, in bands of 8 tile rows with the row index fastest, so that the tiles in flight on
// one XCD share rows of A and of B in its L2
__device__ __forceinline__ void i8_tile(int id, int n, int tm, int tn, int& im, int& in) {
    const int t = i8_xcd(id, n), band = t / (8 * tn), r0 = band * 8, h = min(8, tm - r0), u = t - band * 8 * tn;
    in = u / h; im = r0 + u - in * h;
}

template <typename T, int BM, int BN>
__global__ __launch_bounds__(256) void gemm_i8_kernel(const GemmI8Args a, const int tm, const int tn, const int per) {
#ifdef __HIP_DEVICE_COMPILE__      // the host pass needs the launch stub alone
    constexpr int RB = 128, AT = BM * RB, BT = BN * RB, STAGE = AT + BT, NA = AT / 4096, NB = BT / 4096, WM = BM / 64, WN = BN / 64;
    extern __shared__ __attribute__((aligned(16))) char lds_i8[];
    const int tid = threadIdx.x, lane = tid & 63, ml = lane & 31, kl = lane >> 5;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6), wr = wave >> 1, wc = wave & 1;
    int im, in;
    i8_tile(blockIdx.x, gridDim.x, tm, tn, im, in);
    const int m0 = im * BM, n0 = in * BN, split = blockIdx.y;
    const __amdgpu_buffer_rsrc_t srdA = i8_srd(a.A + (long)m0 * a.lda), srdB = i8_srd(a.B + (long)n0 * a.ldb);
    int ao[NA], bo[NB], kc[NA > NB ? NA : NB];
#pragma unroll
    for (int i = 0; i < (NA > NB ? NA : NB); ++i) {
        const int idx = tid + 256 * i, r = idx >> 3, c = ((idx & 7) ^ ((r >> 1) & 7)) * 16;
        kc[i] = c;
        if (i < NA) ao[i] = m0 + r < a.M ? (int)((long)r * a.lda + c) : I8_OOB;
        if (i < NB) bo[i] = n0 + r < a.N ? (int)((long)r * a.ldb + c) : I8_OOB;
    }
    const int t0 = split * per, t1 = min((a.K + RB - 1) / RB, t0 + per), wbase = wave * 1024;
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
    if (t0 < t1) stage(t0);
    for (int t = t0; t < t1; ++t) {
        asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
        __builtin_amdgcn_s_barrier();
        asm volatile("" ::: "memory");
        if (t + 1 < t1) stage(t + 1);
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
    __syncthreads();                                             // the ring is idle: each wave parks its sums in its own part of it
    int* S = reinterpret_cast<int*>(lds_i8) + wave * (BM / 2) * (BN / 2);
#pragma unroll
    for (int i = 0; i < WM; ++i)
#pragma unroll
        for (int j = 0; j < WN; ++j)
#pragma unroll
            for (int r = 0; r < 16; ++r) S[(i * 32 + (r & 3) + 8 * (r >> 2) + 4 * kl) * (BN / 2) + j * 32 + ml] = acc[i][j][r];
    asm volatile("" ::: "memory");
    i8_finish<T, BM / 2, BN / 2>(a, S, m0 + wr * (BM / 2), n0 + wc * (BN / 2), lane, i8_aligned<T>(a), a.nsplit > 1 ? a.part + (long)split * a.M * a.N : nullptr);
#endif
}
// adds the parts of a split K axis and finishes the outputs; 4 columns a thread
template <typename T>
__global__ __launch_bounds__(256) void gemm_i8_sum_kernel(const GemmI8Args a) {
    const long mn = (long)a.M * a.N, i = ((long)blockIdx.x * 256 + threadIdx.x) * 4;
    if (i >= mn) return;
    int v[4] = {0, 0, 0, 0};
    if (mn % 4 == 0) {
        for (int s = 0; s < a.nsplit; ++s) {
            const i32x4 x = *reinterpret_cast<const i32x4*>(a.part + s * mn + i);
            v[0] += x[0]; v[1] += x[1]; v[2] += x[2]; v[3] += x[3];
        }
    } else {
        for (int s = 0; s < a.nsplit; ++s)
            for (int e = 0; e < 4; ++e) if (i + e < mn) v[e] += a.part[s * mn + i + e];
    }
    for (int e = 0; e < 4; ++e) if (i + e < mn) i8_put<T>(a, v[e], (int)((i + e) / a.N), (int)((i + e) % a.N));
}

// ---------------------------------------------------------------- few tokens
// MT x 16 tokens, NT x 16 weight rows a block; lane (l15, g) of a step of 64 k holds bytes 16g .. 16g+15 of row l15 of both operands. The
// accumulator has the weight row in its registers (4g + r) and the token in its lane (l15).
constexpr int FEW_W = 8;                                         // waves: parts of K
template <typename T, int MT, int NT>
__global__ __launch_bounds__(512) void gemm_i8_few_kernel(const GemmI8Args a) {
#ifdef __HIP_DEVICE_COMPILE__
    __shared__ __attribute__((aligned(16))) int red[FEW_W][NT * 16 * MT * 16 + 4];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), l15 = lane & 15, g = lane >> 4;
    const int n0 = blockIdx.x * (16 * NT);
    const int steps = (a.K + 63) / 64, per = (steps + FEW_W - 1) / FEW_W, s0 = min(wave * per, steps), s1 = min(s0 + per, steps);
    const int8_t *wp[NT], *ap[MT];
#pragma unroll
    for (int j = 0; j < NT; ++j) wp[j] = a.B + (long)min(n0 + 16 * j + l15, a.N - 1) * a.ldb + 16 * g;      // rows past the end: any row, dropped
#pragma unroll
    for (int i = 0; i < MT; ++i) ap[i] = a.A + (long)min(16 * i + l15, a.M - 1) * a.lda + 16 * g;
    i32x4 acc[MT][NT];
#pragma unroll
    for (int i = 0; i < MT; ++i)
#pragma unroll
        for (int j = 0; j < NT; ++j) acc[i][j] = (i32x4){0, 0, 0, 0};
    constexpr int UN = NT == 1 ? 4 : 2;                          // steps whose loads are in flight together
    int s = s0;
    for (; s + UN <= s1 && (s + UN) * 64 <= a.K; s += UN) {
        i32x4 w[UN][NT], x[UN][MT];
#pragma unroll
        for (int u = 0; u < UN; ++u) {
#pragma unroll
            for (int j = 0; j < NT; ++j) w[u][j] = *reinterpret_cast<const i32x4*>(wp[j] + (s + u) * 64);
#pragma unroll
            for (int i = 0; i < MT; ++i) x[u][i] = *reinterpret_cast<const i32x4*>(ap[i] + (s + u) * 64);
        }
#pragma unroll
        for (int u = 0; u < UN; ++u)
#pragma unroll
            for (int i = 0; i < MT; ++i)
#pragma unroll
                for (int j = 0; j < NT; ++j) acc[i][j] = __builtin_amdgcn_mfma_i32_16x16x64_i8(w[u][j], x[u][i], acc[i][j], 0, 0, 0);
    }
    for (; s < s1; ++s) {                                        // remaining steps, the last of which may end inside
        const bool in = s * 64 + 16 * g < a.K;
        i32x4 w[NT], x[MT];
#pragma unroll
        for (int j = 0; j < NT; ++j) { w[j] = (i32x4){0, 0, 0, 0}; if (in) w[j] = *reinterpret_cast<const i32x4*>(wp[j] + s * 64); }
#pragma unroll
        for (int i = 0; i < MT; ++i) { x[i] = (i32x4){0, 0, 0, 0}; if (in) x[i] = *reinterpret_cast<const i32x4*>(ap[i] + s * 64); }
#pragma unroll
        for (int i = 0; i < MT; ++i)
#pragma unroll
            for (int j = 0; j < NT; ++j) acc[i][j] = __builtin_amdgcn_mfma_i32_16x16x64_i8(w[j], x[i], acc[i][j], 0, 0, 0);
    }
#pragma unroll
    for (int i = 0; i < MT; ++i)
#pragma unroll
        for (int j = 0; j < NT; ++j) *reinterpret_cast<i32x4*>(&red[wave][((16 * i + l15) * NT + j) * 16 + 4 * g]) = acc[i][j];
    __syncthreads();
    for (int e = tid; e < MT * 16 * NT * 16; e += 512) {
        const int m = e / (16 * NT), n = n0 + e - m * (16 * NT);
        int v = 0;
#pragma unroll
        for (int w = 0; w < FEW_W; ++w) v += red[w][e];
        if (m < a.M && n < a.N) i8_put<T>(a, v, m, n);
    }
#endif
}

// ---------------------------------------------------------------- 256 x 256, four phases a k-tile
// The schedule, its hazards and the counted wait are those of cb_gemm_bf16_p8.hip (WM = 2): the two wave groups run one barrier apart, LDS-DMA
// pieces stay in flight over the barriers, and one `s_waitcnt vmcnt(4)` a k-tile retires the tile that comes next. Pieces past the end of K
// are issued all the same, with out-of-range offsets, so that the count holds; the build refuses this file's kernel if it spills.
constexpr int P8_RB = 128, P8_HALF = 128 * P8_RB, P8_TILE = 256 * P8_RB, P8_STAGE = 2 * P8_TILE, P8_LDS = 2 * P8_STAGE;
#define I8_BARRIER() do { asm volatile("" ::: "memory"); __builtin_amdgcn_sched_barrier(0); __builtin_amdgcn_s_barrier(); __builtin_amdgcn_sched_barrier(0); asm volatile("" ::: "memory"); } while (0)
template <typename T>
__global__ __launch_bounds__(512) void gemm_i8_p8_kernel(const GemmI8Args a, const int tm, const int tn) {
#ifdef __HIP_DEVICE_COMPILE__
    extern __shared__ __attribute__((aligned(16))) char lds_i8[];
    char* lds = lds_i8;
    const int tid = threadIdx.x, lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6), wr = wave >> 2, wc = wave & 3;
    int im, in;
    i8_tile(blockIdx.x, gridDim.x, tm, tn, im, in);
    const int m0 = im * 256, n0 = in * 256;
    const int nk = (a.K + P8_RB - 1) / P8_RB;
    int ao[2][2], bo[2][2], kc[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const int idx = tid + i * 512, row = idx >> 3;
        kc[i] = ((idx & 7) ^ ((row >> 1) & 7)) * 16;
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const int r = h * 128 + row;
            ao[h][i] = m0 + r < a.M ? (int)((long)r * a.lda + kc[i]) : I8_OOB;
            bo[h][i] = n0 + r < a.N ? (int)((long)r * a.ldb + kc[i]) : I8_OOB;
        }
    }
    const __amdgpu_buffer_rsrc_t srdA = i8_srd(a.A + (long)m0 * a.lda), srdB = i8_srd(a.B + (long)n0 * a.ldb);
    const int wbase = wave * 1024;
    auto stageA = [&](int t, int h) {
        char* d = lds + (t & 1) * P8_STAGE + h * P8_HALF + wbase;
        const int k0 = t * P8_RB;
#pragma unroll
        for (int i = 0; i < 2; ++i)
            __builtin_amdgcn_raw_ptr_buffer_load_lds(srdA, (lds_vp)(d + i * 8192), 16, k0 + kc[i] < a.K ? ao[h][i] : I8_OOB, k0, 0, 0);
    };
    auto stageB = [&](int t, int h) {
        char* d = lds + (t & 1) * P8_STAGE + P8_TILE + h * P8_HALF + wbase;
        const int k0 = t * P8_RB;
#pragma unroll
        for (int i = 0; i < 2; ++i)
            __builtin_amdgcn_raw_ptr_buffer_load_lds(srdB, (lds_vp)(d + i * 8192), 16, k0 + kc[i] < a.K ? bo[h][i] : I8_OOB, k0, 0, 0);
    };
    i32x16 acc[4][2];
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < 2; ++j)
#pragma unroll
            for (int r = 0; r < 16; ++r) acc[i][j][r] = 0;
    const int kl = lane >> 5, ml = lane & 31, sw = (ml >> 1) & 7;
    const int aoff = (wr * 128 + ml) * P8_RB, boff = P8_TILE + (wc * 64 + ml) * P8_RB;
    int co[4];
#pragma unroll
    for (int s = 0; s < 4; ++s) co[s] = ((2 * s + kl) ^ sw) * 16;
    stageB(0, 0); stageB(0, 1); stageA(0, 0); stageA(0, 1); stageB(1, 0); stageB(1, 1);
    asm volatile("s_waitcnt vmcnt(4)" ::: "memory");
    I8_BARRIER();
    if (wr == 1) I8_BARRIER();                                   // the second group runs one barrier behind the first
    i32x4 av[2][4], b0[4], b1[4];
    auto rd_b = [&](const char* p, i32x4 (&b)[4]) {
#pragma unroll
        for (int s = 0; s < 4; ++s) b[s] = *reinterpret_cast<const i32x4*>(p + co[s]);
    };
    auto rd_a = [&](const char* p, int i0) {
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
            for (int s = 0; s < 4; ++s) av[i][s] = *reinterpret_cast<const i32x4*>(p + (i0 + i) * 32 * P8_RB + co[s]);
    };
    auto mm = [&](int i0, int j, const i32x4 (&b)[4]) {
        __builtin_amdgcn_s_setprio(1);
#pragma unroll
        for (int s = 0; s < 4; ++s)
#pragma unroll
            for (int i = 0; i < 2; ++i) acc[i0 + i][j] = __builtin_amdgcn_mfma_i32_32x32x32_i8(av[i][s], b[s], acc[i0 + i][j], 0, 0, 0);
        __builtin_amdgcn_s_setprio(0);
    };
    auto tile = [&](int t, auto bufc) {
        constexpr int buf = decltype(bufc)::value;
        const char* ab = lds + buf * P8_STAGE + aoff;
        const char* bb = lds + buf * P8_STAGE + boff;
        rd_b(bb, b0); rd_b(bb + 32 * P8_RB, b1); rd_a(ab, 0);
        stageA(t + 1, 0);
        I8_BARRIER();
        mm(0, 0, b0);
        I8_BARRIER();
        stageA(t + 1, 1);
        I8_BARRIER();
        mm(0, 1, b1);
        I8_BARRIER();
        rd_a(ab, 2);
        stageB(t + 2, 0);
        I8_BARRIER();
        mm(2, 1, b1);
        I8_BARRIER();
        stageB(t + 2, 1);
        asm volatile("s_waitcnt vmcnt(4)" ::: "memory");         // k-tile t + 1 is complete; the B halves of t + 2 stay in flight
        I8_BARRIER();
        mm(2, 0, b0);
        I8_BARRIER();
    };
    int t = 0;
    for (; t + 1 < nk; t += 2) { tile(t, std::integral_constant<int, 0>{}); tile(t + 1, std::integral_constant<int, 1>{}); }
    if (t < nk) tile(t, std::integral_constant<int, 0>{});
    if (wr == 0) I8_BARRIER();
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");             // the pieces issued past the end of K
    __syncthreads();
    const bool al = i8_aligned<T>(a);
    int* S = reinterpret_cast<int*>(lds) + wave * (64 * 64);
#pragma unroll
    for (int hf = 0; hf < 2; ++hf) {
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
            for (int j = 0; j < 2; ++j)
#pragma unroll
                for (int r = 0; r < 16; ++r) S[(i * 32 + (r & 3) + 8 * (r >> 2) + 4 * kl) * 64 + j * 32 + ml] = acc[2 * hf + i][j][r];
        asm volatile("" ::: "memory");
        i8_finish<T, 64, 64>(a, S, m0 + wr * 128 + hf * 64, n0 + wc * 64, lane, al, nullptr);
        asm volatile("" ::: "memory");
    }
#endif
}

// ---------------------------------------------------------------- host side
enum { I8_FEW = 0, I8_64 = 1, I8_128 = 2, I8_256 = 3 };
struct I8Plan { int kind = I8_64, nsplit = 1, per = 0; };
static I8Plan i8_plan(const GemmI8Args& a) {
    I8Plan p;
    const long t256 = (long)cdiv(a.M, 256) * cdiv(a.N, 256), t128 = (long)cdiv(a.M, 128) * cdiv(a.N, 128), t64 = (long)cdiv(a.M, 64) * cdiv(a.N, 64);
    const int nk = (int)cdiv(a.K, 128);
    p.per = nk;
    // All figures in us, replayed from a graph, weights not in cache. Few tokens: the kernel for them reads the tokens once per 16 weight rows, so it
    // is taken up to 64 tokens and M N K = 1.5 x 2^30; it / the 64 tile: M N K = 2^26.6 (17 tokens, 2304 x 768) 3.4 / 6.3, 2^29 (32, 4096 x 4096)
    // 8.8 / 15.3, 2^30 (16, 8192 x 8192) 18.2 / 21.4, 1.5 x 2^30 (16, 24576 x 4096) 28.0 / 30.6, 2^31 (64, 8192 x 4096) 17.8 / 19.7 but (32, 8192 x
    // 8192) 26.2 / 22.6, 2^32 (64, 4096 x 16384) 50.6 / 27.5
    if (a.M <= 64 && (long)a.M * a.N * a.K <= 3L << 29) { p.kind = I8_FEW; return p; }
    // 256 against 128 tiles (us of a call): 128 of them (1024 x 8192 x 4096) 48.4 / 41.1, 160 (2560 x 4096 x 4096) 50.8 / 60.1, 196 (3584 x 3584 x
    // 4096) 55.0 / 70.4. Only where a tile's rows are more than half there: 192 tiles of N = 49152, K = 4096 with 128 rows 56.3 / 52.0, with 129 57.4 / 74.0
    if (t256 >= 160 && a.M > 128) { p.kind = I8_256; return p; }
    // 128 against 64 tiles: 192 of them (128 x 24576 x 4096) 68 / 34, 256 (512 x 8192 x 4096) 33.8 / 35.2, (512 x 8192 x 8192) 61 / 66, 384 (256 x 24576
    // x 4096) 45.6 / 62. With rows enough for both: N = 49152, K = 4096, 64 rows 47.8 / 43.3, 65 rows 47.6 / 61.4; N = 40960, K = 2048 25.2 / 20.4, 25.0 / 32.2
    p.kind = t128 >= 256 && a.M > 64 ? I8_128 : I8_64;
    const long t = p.kind == I8_128 ? t128 : t64;
    // fewer tiles than CUs: K is split into runs of at least 8 k-tiles for two blocks a CU. 64 x 4096 x 4096 (64 tiles) whole / 4 runs of 8 / 8 of 4:
    // 26.0 / 17.9 / 20.9; 64 x 8192 x 8192 (128 tiles) whole / 4 / 8: 50 / 26 / 31. As many 64 tiles as CUs: four runs where K is long (128 x 8192 x 8192
    // 49 / 38, 256 x 4096 x 16384 88 / 53), none where it is not (128 x 8192 x 4096 25.7 / 28.9)
    const long runs = t < 256 ? cdiv(512, t) : p.kind == I8_64 && t == 256 && nk >= 64 ? 4 : 1;
    if (runs > 1 && nk >= 16) {
        p.nsplit = (int)std::min<long>(runs, nk / 8);
        p.per = (int)cdiv(nk, p.nsplit);
        p.nsplit = (int)cdiv(nk, p.per);
    }
    return p;
}
size_t gemm_i8_ws_bytes(const GemmI8Args& a) {
    const I8Plan p = i8_plan(a);
    return p.nsplit > 1 ? (size_t)p.nsplit * a.M * a.N * 4 : 0;
}
template <typename T, int BM, int BN> static void i8_go(const Launch& L, const GemmI8Args& a, const I8Plan& p) {
    const int tm = (int)cdiv(a.M, BM), tn = (int)cdiv(a.N, BN);
    constexpr int lds = 2 * (BM + BN) * 128;
    static_assert(lds >= BM * BN * 4, "the sums are parked in the ring");
    set_dyn_lds(reinterpret_cast<const void*>(&gemm_i8_kernel<T, BM, BN>), 160 * 1024);
    hipLaunchKernelGGL((gemm_i8_kernel<T, BM, BN>), dim3((unsigned)tm * tn, p.nsplit), dim3(256), lds, L.stream, a, tm, tn, p.per);
}
template <typename T> static void i8_any(const Launch& L, GemmI8Args a, void* ws) {
    const I8Plan p = i8_plan(a);
    a.nsplit = p.nsplit;
    a.part = static_cast<int*>(ws);
    const long bm = p.kind == I8_256 ? 256 : p.kind == I8_128 ? 128 : 64;
    const long threads = p.kind == I8_FEW ? 512l * cdiv(a.N, a.M <= 32 ? 16 : 32) : (p.kind == I8_256 ? 512l : 256l) * cdiv(a.M, bm) * cdiv(a.N, bm);
    CB_CHECK(threads < (1l << 32), CB_ERR_SHAPE, "gemm_i8: %d x %d outputs are too many for one call", a.M, a.N);
    L.count(p.nsplit > 1 ? 2 : 1);
    if (L.stats) { L.stats->gemm_flops += 2.0 * a.M * a.N * (double)a.K; L.stats->gemm_launches++; }
    if (L.dry) return;
    if (p.kind == I8_FEW) {
        if (a.M <= 16) hipLaunchKernelGGL((gemm_i8_few_kernel<T, 1, 1>), dim3(cdiv(a.N, 16)), dim3(512), 0, L.stream, a);
        else if (a.M <= 32) hipLaunchKernelGGL((gemm_i8_few_kernel<T, 2, 1>), dim3(cdiv(a.N, 16)), dim3(512), 0, L.stream, a);
        else hipLaunchKernelGGL((gemm_i8_few_kernel<T, 4, 2>), dim3(cdiv(a.N, 32)), dim3(512), 0, L.stream, a);
    } else if (p.kind == I8_256) {
        const int tm = (int)cdiv(a.M, 256), tn = (int)cdiv(a.N, 256);
        set_dyn_lds(reinterpret_cast<const void*>(&gemm_i8_p8_kernel<T>), P8_LDS);
        hipLaunchKernelGGL((gemm_i8_p8_kernel<T>), dim3((unsigned)tm * tn), dim3(512), P8_LDS, L.stream, a, tm, tn);
    } else if (p.kind == I8_128) i8_go<T, 128, 128>(L, a, p);
    else i8_go<T, 64, 64>(L, a, p);
    CB_HIP(hipGetLastError());
    if (p.nsplit > 1) {
        hipLaunchKernelGGL((gemm_i8_sum_kernel<T>), dim3(cdiv((long)a.M * a.N, 1024)), dim3(256), 0, L.stream, a);
        CB_HIP(hipGetLastError());
    }
}
void gemm_i8(const Launch& L, const GemmI8Args& a, void* ws) { CB_DT_SWITCH(a.dt, T, i8_any<T>(L, a, ws)); }

}  // namespace cb
