// cb_norm_i8.hip — root-mean-square norm with the residual's addition, in its element type or in 8 bits with a scale per row, its backward
// pass, and plain rows brought to 8 bits.
//
//   h = round_T(x + r)          the residual stream as it is held; everything below is of the held value
//   rstd = 1 / sqrt(mean(h^2) + eps);  y = h rstd g
//   8 bits: scale = max|y| / 127, q = rint(y * (127 / max|y|))    (of the unrounded y)
//   dh = rstd (dy g - h rstd^2 mean(dy g h)) + dres;  dg = sum over rows of dy h rstd
// All of it is bound by memory: a row is read once and stays in registers (8 consecutive elements a thread and step) until it is written.
#include "cb_device.h"
#include "cb_i8.h"

namespace cb {

template <typename T> __device__ __forceinline__ void ld8v(const T* p, float (&v)[8]) {
    const float4 a = ld4(p), b = ld4(p + 4);
    v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w; v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
}
template <> __device__ __forceinline__ void ld8v<bf16_t>(const bf16_t* p, float (&v)[8]) {
    const bf16x8_t t = *reinterpret_cast<const bf16x8_t*>(p);
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = (float)t[e];
}
template <typename T> __device__ __forceinline__ void st8v(T* p, const float (&v)[8]) {
    st4(p, make_float4(v[0], v[1], v[2], v[3])); st4(p + 4, make_float4(v[4], v[5], v[6], v[7]));
}
template <> __device__ __forceinline__ void st8v<bf16_t>(bf16_t* p, const float (&v)[8]) {
    bf16x8_t o;
#pragma unroll
    for (int e = 0; e < 8; ++e) o[e] = (bf16_t)v[e];
    *reinterpret_cast<bf16x8_t*>(p) = o;
}
// 8 elements of a row from column c on; VEC: rows of whole, aligned groups of 8. Elements at or beyond C are 0
template <typename T, bool VEC> __device__ __forceinline__ void row_ld(const T* p, int c, int C, float (&v)[8]) {
    if constexpr (VEC) {
        if (c < C) { ld8v(p + c, v); return; }
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = 0.f;
    } else {
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = c + e < C ? ld1(p + c + e) : 0.f;
    }
}
template <typename T, bool VEC> __device__ __forceinline__ void row_st(T* p, int c, int C, const float (&v)[8]) {
    if constexpr (VEC) {
        if (c < C) st8v(p + c, v);
    } else {
#pragma unroll
        for (int e = 0; e < 8; ++e) if (c + e < C) st1(p + c + e, v[e]);
    }
}
// sums / maxima over the TPR threads of a row (64: a wave; 256: the block), the same value in all of them
template <int TPR> __device__ __forceinline__ float row_sum(float v, float* sh) {
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) v += __shfl_xor(v, o, 64);
    if constexpr (TPR == 256) {
        __syncthreads();
        if ((threadIdx.x & 63) == 0) sh[threadIdx.x >> 6] = v;
        __syncthreads();
        v = (sh[0] + sh[1]) + (sh[2] + sh[3]);
    }
    return v;
}
template <int TPR> __device__ __forceinline__ unsigned row_max(unsigned v, float* sh) {
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) v = max(v, (unsigned)__shfl_xor((int)v, o, 64));
    if constexpr (TPR == 256) {
        unsigned* s = reinterpret_cast<unsigned*>(sh);
        __syncthreads();
        if ((threadIdx.x & 63) == 0) s[threadIdx.x >> 6] = v;
        __syncthreads();
        v = max(max(s[0], s[1]), max(s[2], s[3]));
    }
    return v;
}
// the factor 127 / amax of a row and the scale that it is held with. Magnitudes are compared as bit patterns, so that a NaN or an infinity is
// the largest: such a row gets that as its scale and zeros as its values. A row below 2^-119 (127 / amax would overflow) is held as zeros.
__device__ __forceinline__ float i8_factor(unsigned amax_bits, float* scale) {
    const float amax = __uint_as_float(amax_bits);
    if (amax_bits >= 0x7F800000u) { *scale = amax; return 0.f; }
    if (amax < 1.5e-36f) { *scale = 0.f; return 0.f; }
    *scale = amax / 127.f;
    return 127.f / amax;
}
__device__ __forceinline__ unsigned mag(float v) { return __float_as_uint(v) & 0x7FFFFFFFu; }
__device__ __forceinline__ int i8_of(float v, float f) { return f == 0.f ? 0 : (int)fminf(fmaxf(rintf(v * f), -127.f), 127.f); }
// 8 values to q[c .. c+7] of a row of Cp = ceil16(C) places (the row is 16-byte aligned)
__device__ __forceinline__ void i8_store(int8_t* q, int c, int Cp, const float (&v)[8], float f) {
    if (c >= Cp) return;
    int b[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) b[e] = i8_of(v[e], f) & 255;
    *reinterpret_cast<uint2*>(q + c) = make_uint2((unsigned)(b[0] | (b[1] << 8) | (b[2] << 16) | (b[3] << 24)), (unsigned)(b[4] | (b[5] << 8) | (b[6] << 16) | (b[7] << 24)));
}

// NORM = false: rows to 8 bits as they are
template <typename T, int TPR, int NV, bool VEC, bool NORM>
__global__ __launch_bounds__(256) void rms_fwd_kernel(const RmsArgs a) {
    __shared__ float sh[4];
    const long row = (long)blockIdx.x * (256 / TPR) + threadIdx.x / TPR;
    if (row >= a.rows) return;                       // TPR = 256: the whole block
    const int t = threadIdx.x % TPR, C = a.C;
    const T* x = static_cast<const T*>(a.x) + row * a.ldx;
    float v[NV][8];
#pragma unroll
    for (int j = 0; j < NV; ++j) row_ld<T, VEC>(x, (j * TPR + t) * 8, C, v[j]);
    if constexpr (NORM) {
        if (a.r) {
            const T* r = static_cast<const T*>(a.r) + row * a.ldr;
#pragma unroll
            for (int j = 0; j < NV; ++j) {
                float w[8];
                row_ld<T, VEC>(r, (j * TPR + t) * 8, C, w);
#pragma unroll
                for (int e = 0; e < 8; ++e) v[j][e] = (float)(T)(v[j][e] + w[e]);
            }
        }
        if (a.h) {
            T* h = static_cast<T*>(a.h) + row * a.ldh;
#pragma unroll
            for (int j = 0; j < NV; ++j) row_st<T, VEC>(h, (j * TPR + t) * 8, C, v[j]);
        }
        float ss = 0.f;
#pragma unroll
        for (int j = 0; j < NV; ++j) {
            float s = 0.f;
#pragma unroll
            for (int e = 0; e < 8; ++e) s = __builtin_fmaf(v[j][e], v[j][e], s);
            ss += s;
        }
        const float ms = row_sum<TPR>(ss, sh) / (float)C;
        float rstd = 1.f / sqrtf(ms + a.eps);
        // squares beyond fp32's range, or so small that they lost bits beside no greater eps: once more, of the row times 2^-100 or 2^100
        if (!(ms < 3e38f) || ms + a.eps < 0x1p-90f) {
            const float f = ms + a.eps < 0x1p-90f ? 0x1p100f : 0x1p-100f;
            ss = 0.f;
#pragma unroll
            for (int j = 0; j < NV; ++j)
#pragma unroll
                for (int e = 0; e < 8; ++e) { const float x = v[j][e] * f; ss = __builtin_fmaf(x, x, ss); }
            rstd = f / sqrtf(row_sum<TPR>(ss, sh) / (float)C + a.eps * f * f);
        }
        if (t == 0 && a.rstd) a.rstd[row] = rstd;
#pragma unroll
        for (int j = 0; j < NV; ++j) {
            const int c = (j * TPR + t) * 8;
            float g[8];
            row_ld<float, VEC>(a.gamma, c, C, g);
#pragma unroll
            for (int e = 0; e < 8; ++e) v[j][e] = v[j][e] * rstd * g[e];
        }
        if (a.y) {
            T* y = static_cast<T*>(a.y) + row * a.ldy;
#pragma unroll
            for (int j = 0; j < NV; ++j) row_st<T, VEC>(y, (j * TPR + t) * 8, C, v[j]);
            return;
        }
    }
    unsigned m = 0;
#pragma unroll
    for (int j = 0; j < NV; ++j)
#pragma unroll
        for (int e = 0; e < 8; ++e) m = max(m, mag(v[j][e]));
    float s;
    const float f = i8_factor(row_max<TPR>(m, sh), &s);
    if (t == 0) a.scale[row] = s;
    int8_t* q = a.q + row * a.ldq;
    const int Cp = (C + 15) / 16 * 16;
#pragma unroll
    for (int j = 0; j < NV; ++j) i8_store(q, (j * TPR + t) * 8, Cp, v[j], f);
}
// rows longer than the registers hold: read twice (the second time from the caches)
template <typename T>
__global__ __launch_bounds__(256) void quantize_long_kernel(const RmsArgs a) {
    __shared__ float sh[4];
    const long row = blockIdx.x;
    const T* x = static_cast<const T*>(a.x) + row * a.ldx;
    const int C = a.C, Cp = (C + 15) / 16 * 16;
    unsigned m = 0;
    for (int c = threadIdx.x; c < C; c += 256) m = max(m, mag(ld1(x + c)));
    float s;
    const float f = i8_factor(row_max<256>(m, sh), &s);
    if (threadIdx.x == 0) a.scale[row] = s;
    int8_t* q = a.q + row * a.ldq;
    for (int c = threadIdx.x; c < Cp; c += 256) q[c] = c < C ? (int8_t)i8_of(ld1(x + c), f) : (int8_t)0;
}

// blocks of the backward pass, and rows of its partial sums of dgamma. 16384 x 2048 bf16, blocks 512 / 768 / 1024 / 2048: 86 / 67 / 57 / 60 us
// (57 us: 277 MB at 4.9 TB/s, what a copy reaches) + 5 / 6 / 5 / 8 us for the join; a wave a row instead of a block 80 us at 512
constexpr int RMS_PARTS = 1024;
template <typename T, int TPR, int NV, bool VEC>
__global__ __launch_bounds__(256) void rms_bwd_kernel(const RmsArgs a, const int per) {
    __shared__ float sh[4];
    __shared__ float dgs[TPR == 64 ? NV * 64 * 8 : 8];
    const int t = threadIdx.x % TPR, sub = threadIdx.x / TPR, C = a.C;
    constexpr int RPB = 256 / TPR;
    float g[NV][8], dg[NV][8];
#pragma unroll
    for (int j = 0; j < NV; ++j) {
        row_ld<float, VEC>(a.gamma, (j * TPR + t) * 8, C, g[j]);
#pragma unroll
        for (int e = 0; e < 8; ++e) dg[j][e] = 0.f;
    }
    const long r0 = (long)blockIdx.x * per, r1 = min(r0 + per, a.rows);
    for (long row = r0 + sub; row < r1; row += RPB) {
        const T* hp = static_cast<const T*>(a.h) + row * a.ldh;
        const T* dp = static_cast<const T*>(a.dy) + row * a.lddy;
        const float rstd = a.rstd[row];
        const T* dr = a.dres ? static_cast<const T*>(a.dres) + row * a.lddres : nullptr;
        float h[NV][8], w[NV][8], o[NV][8], s = 0.f;
#pragma unroll
        for (int j = 0; j < NV; ++j) {
            row_ld<T, VEC>(hp, (j * TPR + t) * 8, C, h[j]);
            row_ld<T, VEC>(dp, (j * TPR + t) * 8, C, w[j]);
            if (dr) row_ld<T, VEC>(dr, (j * TPR + t) * 8, C, o[j]);
        }
#pragma unroll
        for (int j = 0; j < NV; ++j)
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                h[j][e] *= rstd;                                   // normed value
                dg[j][e] = __builtin_fmaf(w[j][e], h[j][e], dg[j][e]);
                w[j][e] *= g[j][e];
                s = __builtin_fmaf(w[j][e], h[j][e], s);
            }
        const float m = row_sum<TPR>(s, sh) / (float)C;
        T* dh = static_cast<T*>(a.dh) + row * a.lddh;
#pragma unroll
        for (int j = 0; j < NV; ++j) {
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const float v = rstd * (w[j][e] - h[j][e] * m);
                o[j][e] = dr ? v + o[j][e] : v;
            }
            row_st<T, VEC>(dh, (j * TPR + t) * 8, C, o[j]);
        }
    }
    if (!a.part) return;
    float* P = a.part + (long)blockIdx.x * C;
    if constexpr (TPR == 256) {
#pragma unroll
        for (int j = 0; j < NV; ++j) row_st<float, false>(P, (j * TPR + t) * 8, C, dg[j]);
    } else {
        for (int k = 0; k < RPB; ++k) {                            // one wave after the other: a fixed order
            if (sub == k) {
#pragma unroll
                for (int j = 0; j < NV; ++j)
#pragma unroll
                    for (int e = 0; e < 8; ++e) {
                        const int i = (j * 64 + t) * 8 + e;
                        dgs[i] = k ? dgs[i] + dg[j][e] : dg[j][e];
                    }
            }
            __syncthreads();
        }
        for (int c = threadIdx.x; c < C; c += 256) P[c] = dgs[c];
    }
}
// dgamma[c] = sum of the parts in a fixed order: 16 columns a block (one 64-byte piece of a part), 16 runs of parts joined in LDS
__global__ __launch_bounds__(256) void rms_dgamma_kernel(const float* __restrict__ part, float* __restrict__ dgamma, int n, int C) {
    __shared__ float sh[16][17];
    const int x = threadIdx.x & 15, w = threadIdx.x >> 4, c = blockIdx.x * 16 + x;
    float s = 0.f;
    if (c < C) {
#pragma unroll 8
        for (int i = w; i < n; i += 16) s += part[(long)i * C + c];
    }
    sh[w][x] = s;
    __syncthreads();
    if (w == 0 && c < C) {
        float t = 0.f;
#pragma unroll
        for (int i = 0; i < 16; ++i) t += sh[i][x];
        dgamma[c] = t;
    }
}

// ---------------------------------------------------------------- host side
static bool al16(const void* p, long ld, size_t es) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0 && ld * (long)es % 16 == 0; }
#define RMS_GO(kernel, grid, ...)                                                        \
    do {                                                                                 \
        L.count();                                                                       \
        if (!L.dry) {                                                                    \
            hipLaunchKernelGGL(kernel, dim3(grid), dim3(256), 0, L.stream, __VA_ARGS__); \
            CB_HIP(hipGetLastError());                                                   \
        }                                                                                \
    } while (0)
// threads a row and groups of 8 a thread: a wave up to 1024 columns, else a block. Forward with a residual, bf16, 33.5 M elements, a wave / a block a row:
// 512 columns 39.8 / 67.7 us, 1024 39.1 / 45.5, 2048 43.1 / 39.4, 4096 44.9 / 40.6
#define RMS_SHAPE(C, TPR, NV, ...)                                                            \
    do {                                                                                      \
        if ((C) <= 512) { constexpr int TPR = 64, NV = 1; __VA_ARGS__; }                      \
        else if ((C) <= 1024) { constexpr int TPR = 64, NV = 2; __VA_ARGS__; }                \
        else if ((C) <= 2048) { constexpr int TPR = 256, NV = 1; __VA_ARGS__; }               \
        else if ((C) <= 4096) { constexpr int TPR = 256, NV = 2; __VA_ARGS__; }               \
        else if ((C) <= 8192) { constexpr int TPR = 256, NV = 4; __VA_ARGS__; }               \
        else { constexpr int TPR = 256, NV = 8; __VA_ARGS__; }                                \
    } while (0)

// backward: a wave up to 512 columns, else a block (a row's gradient, norm and gamma parts would take a wave over 200 registers)
#define RMS_BWD_SHAPE(C, TPR, NV, ...)                                                        \
    do {                                                                                      \
        if ((C) <= 512) { constexpr int TPR = 64, NV = 1; __VA_ARGS__; }                      \
        else if ((C) <= 2048) { constexpr int TPR = 256, NV = 1; __VA_ARGS__; }               \
        else if ((C) <= 4096) { constexpr int TPR = 256, NV = 2; __VA_ARGS__; }               \
        else if ((C) <= 8192) { constexpr int TPR = 256, NV = 4; __VA_ARGS__; }               \
        else { constexpr int TPR = 256, NV = 8; __VA_ARGS__; }                                \
    } while (0)

template <bool NORM> static void fwd_rows(const Launch& L, const RmsArgs& a) {
    const size_t es = dt_size(a.dt);
    const bool vec = a.C % 8 == 0 && al16(a.x, a.ldx, es) && (!a.r || al16(a.r, a.ldr, es)) && (!a.h || al16(a.h, a.ldh, es)) &&
                     (!a.y || al16(a.y, a.ldy, es)) && (!NORM || al16(a.gamma, 0, 4));
    CB_DT_SWITCH(a.dt, T, RMS_SHAPE(a.C, TPR, NV, {
        const unsigned grid = cdiv(a.rows, 256 / TPR);
        if (vec) RMS_GO((rms_fwd_kernel<T, TPR, NV, true, NORM>), grid, a);
        else RMS_GO((rms_fwd_kernel<T, TPR, NV, false, NORM>), grid, a);
    }));
}
// a launch holds fewer than 2^32 threads a dimension: more rows than 2^23 go in several
template <typename F> static void by_rows(const RmsArgs& a, F&& f) {
    const long most = 1l << 23, es = (long)dt_size(a.dt);
    for (long r0 = 0; r0 < a.rows; r0 += most) {
        RmsArgs b = a;
        b.rows = std::min(most, a.rows - r0);
        b.x = static_cast<const char*>(a.x) + r0 * a.ldx * es;
        if (a.r) b.r = static_cast<const char*>(a.r) + r0 * a.ldr * es;
        if (a.h) b.h = static_cast<char*>(a.h) + r0 * a.ldh * es;
        if (a.y) b.y = static_cast<char*>(a.y) + r0 * a.ldy * es;
        if (a.q) b.q = a.q + r0 * a.ldq;
        if (a.scale) b.scale = a.scale + r0;
        if (a.rstd) b.rstd = a.rstd + r0;
        f(b);
    }
}
void k_rmsnorm_fwd(const Launch& L, const RmsArgs& a) { by_rows(a, [&](const RmsArgs& b) { fwd_rows<true>(L, b); }); }
void k_quantize_rows(const Launch& L, const RmsArgs& a) {
    by_rows(a, [&](const RmsArgs& b) {
        if (b.C <= RMS_MAX_C) fwd_rows<false>(L, b);
        else CB_DT_SWITCH(b.dt, T, RMS_GO((quantize_long_kernel<T>), (unsigned)b.rows, b));
    });
}
static int bwd_per(long rows, int C) {                // rows a block: a whole number of passes of its waves
    const int rpb = C <= 512 ? 4 : 1;
    return (int)rup((long)cdiv(rows, RMS_PARTS), rpb);
}
size_t rmsnorm_bwd_ws_bytes(long rows, int C) { return rows ? (size_t)cdiv(rows, bwd_per(rows, C)) * C * 4 : 0; }
void k_rmsnorm_bwd(const Launch& L, const RmsArgs& a) {
    const size_t es = dt_size(a.dt);
    const bool vec = a.C % 8 == 0 && al16(a.h, a.ldh, es) && al16(a.dy, a.lddy, es) && al16(a.dh, a.lddh, es) && al16(a.gamma, 0, 4) &&
                     (!a.dres || al16(a.dres, a.lddres, es));
    const int per = bwd_per(a.rows, a.C), n = a.rows ? (int)cdiv(a.rows, per) : 0;
    if (n) CB_DT_SWITCH(a.dt, T, RMS_BWD_SHAPE(a.C, TPR, NV, {
        if (vec) RMS_GO((rms_bwd_kernel<T, TPR, NV, true>), (unsigned)n, a, per);
        else RMS_GO((rms_bwd_kernel<T, TPR, NV, false>), (unsigned)n, a, per);
    }));
    if (a.dgamma) RMS_GO(rms_dgamma_kernel, cdiv(a.C, 16), a.part, a.dgamma, n, a.C);
}

}  // namespace cb
