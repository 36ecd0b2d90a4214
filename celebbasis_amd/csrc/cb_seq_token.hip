// cb_seq_token.hip — the attention of cb_seq.h for one new token a sample (Nq = 1): bound by reading the visible keys and values once.
//
// A matrix tile of 16 queries would hold one live row; here a row of K or V is read by PP lanes, 16 bytes each, and multiplied with the (up to
// 8) query heads that share it in registers: dot products close over the PP lanes, everything else stays in the lane. Each group of PP lanes
// has its own keys and its own running maximum, sum and output; groups, waves and blocks are joined once at the end (fixed order). A block has 4
// waves; samples with a long cache are split over blocks by their own length, and seq_combine_kernel joins the parts.
// VALU work per 16 bytes: about 38 + 26 R instructions a lane for R heads, 54 to 10 bytes a clock and CU against the 8 that memory delivers.
#include "cb_seq.h"
#include <algorithm>

namespace cb {

template <int CTRL> __device__ __forceinline__ float tok_dpp(float v) {
    return __int_as_float(__builtin_amdgcn_mov_dpp(__float_as_int(v), CTRL, 0xf, 0xf, false));
}
// sum over aligned groups of PP lanes, in all of them: within 16 lanes by DPP (quad permutes, then mirrors, which after the quads exchange halves)
template <int PP> __device__ __forceinline__ float tok_sum(float v) {
    v += tok_dpp<0xB1>(v);                                       // quad_perm [1,0,3,2]
    v += tok_dpp<0x4E>(v);                                       // quad_perm [2,3,0,1]
    if constexpr (PP >= 8) v += tok_dpp<0x141>(v);               // row_half_mirror
    if constexpr (PP >= 16) v += tok_dpp<0x140>(v);              // row_mirror
    if constexpr (PP >= 32) v += __shfl_xor(v, 16, 64);
    if constexpr (PP >= 64) v += __shfl_xor(v, 32, 64);
    return v;
}
template <typename T> struct TokPiece;
template <> struct TokPiece<bf16_t> {
    static constexpr int E = 8;
    static __device__ __forceinline__ void open(const u32x4s& u, float (&v)[8]) {
#pragma unroll
        for (int i = 0; i < 4; ++i) { v[2 * i] = __uint_as_float(u[i] << 16); v[2 * i + 1] = __uint_as_float(u[i] & 0xffff0000u); }
    }
};
template <> struct TokPiece<float> {
    static constexpr int E = 4;
    static __device__ __forceinline__ void open(const u32x4s& u, float (&v)[4]) {
#pragma unroll
        for (int i = 0; i < 4; ++i) v[i] = __uint_as_float(u[i]);
    }
};

template <typename T, int PP, int R, bool BIAS>
__global__ __launch_bounds__(256) void seq_token_kernel(const SeqArgs a) {
#ifdef __HIP_DEVICE_COMPILE__
    using P = TokPiece<T>;
    constexpr int E = P::E, ROWS = 64 / PP, U = 4, STEP = 4 * ROWS * U;      // keys a block takes a turn
    __shared__ float sm[4][R], sl[4][R];
    __shared__ __attribute__((aligned(16))) float so[4][R][PP * E];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), p = lane % PP, grp = lane / PP;
    const int bk = blockIdx.x, b = bk / a.Hkv, hk = bk - b * a.Hkv, split = blockIdx.y;
    const int pos = seq_pos(a.q_pos, b);
    int kend = seq_clamp_len(a.kv_len, b, a.Nk);
    if (a.causal) kend = max(0, min(kend, pos + 1));
    if (seq_clamp_len(a.q_len, b, 1) < 1) kend = 0;
    int k0 = 0, k1 = kend;
    if (a.nsplit > 1) {
        const int per = ((kend + a.nsplit - 1) / a.nsplit + STEP - 1) / STEP * STEP;
        k0 = min(split * per, kend); k1 = min(k0 + per, kend);
    }
    const bool in = p * E < a.d;                                 // this lane's piece is part of the head dim
    const T* K = static_cast<const T*>(a.k.p) + b * a.k.batch + hk * a.k.head + p * E;
    const T* V = static_cast<const T*>(a.v.p) + b * a.v.batch + hk * a.v.head + p * E;
    const unsigned char* mask = a.mask ? a.mask + b * a.mask_b : nullptr;
    float q[R][E], o[R][E], m[R], l[R], far_l[R], far_r[R];
#pragma unroll
    for (int r = 0; r < R; ++r) {
        const int h = hk * a.G + (r < a.G ? r : 0);
        u32x4s u = {0u, 0u, 0u, 0u};
        if (in && r < a.G) u = *reinterpret_cast<const u32x4s*>(static_cast<const T*>(a.q.p) + b * a.q.batch + h * a.q.head + p * E);
        P::open(u, q[r]);
        m[r] = -INFINITY; l[r] = 0.f; far_l[r] = far_r[r] = 0.f;
#pragma unroll
        for (int e = 0; e < E; ++e) { q[r][e] *= a.scale * SEQ_L2E; o[r][e] = 0.f; }
        if constexpr (BIAS) {
            far_l[r] = seq_bias_of(a, h, -a.D);
            far_r[r] = seq_bias_of(a, h, a.D);
        }
    }
    // the loads of the next turn are in flight while this one is computed
    struct Turn { u32x4s k[U], v[U]; bool ok[U]; } cur, nxt;
    auto load = [&](int t, Turn& w) {
        const bool all = t + ROWS * U <= k1 && !mask;            // wave-uniform
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int key = t + u * ROWS + grp;
            w.ok[u] = all || (key < k1 && (!mask || mask[key] != 0));
            w.k[u] = (u32x4s){0u, 0u, 0u, 0u}; w.v[u] = w.k[u];
            if (w.ok[u] && in) {
                w.k[u] = *reinterpret_cast<const u32x4s*>(K + (long)key * a.k.row);
                w.v[u] = *reinterpret_cast<const u32x4s*>(V + (long)key * a.v.row);
            }
        }
    };
    int t = k0 + wave * (ROWS * U);
    if (t < k1) load(t, cur);
    for (; t < k1; t += STEP) {
        if (t + STEP < k1) load(t + STEP, nxt);
        const bool all = t + ROWS * U <= k1 && !mask;
        float s[U][R];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            float x[E];
            P::open(cur.k[u], x);
#pragma unroll
            for (int r = 0; r < R; ++r) {
                float d = 0.f;
#pragma unroll
                for (int e = 0; e < E; ++e) d = __builtin_fmaf(q[r][e], x[e], d);
                s[u][r] = tok_sum<PP>(d);
            }
        }
        if constexpr (BIAS) {
            const int lo = t - pos, hi = t + ROWS * U - 1 - pos;
            if (hi <= -a.D || lo >= a.D) {
#pragma unroll
                for (int u = 0; u < U; ++u)
#pragma unroll
                    for (int r = 0; r < R; ++r) s[u][r] += hi <= -a.D ? far_l[r] : far_r[r];
            } else {
#pragma unroll
                for (int u = 0; u < U; ++u) {
                    const int rel = min(max(t + u * ROWS + grp - pos, -a.D), a.D);
#pragma unroll
                    for (int r = 0; r < R; ++r) s[u][r] += seq_bias_of(a, hk * a.G + (r < a.G ? r : 0), rel);
                }
            }
        }
        if (!all) {
#pragma unroll
            for (int u = 0; u < U; ++u)
#pragma unroll
                for (int r = 0; r < R; ++r) s[u][r] = cur.ok[u] ? s[u][r] : -INFINITY;
        }
        float f[R];
#pragma unroll
        for (int r = 0; r < R; ++r) {
            const float mx = fmaxf(fmaxf(s[0][r], s[1][r]), fmaxf(s[2][r], s[3][r])), mnew = fmaxf(m[r], mx);
            const float off = mnew == -INFINITY ? 0.f : mnew;
            f[r] = __builtin_amdgcn_exp2f(m[r] - off);            // m = -inf: 0
            m[r] = mnew;
            l[r] *= f[r];
#pragma unroll
            for (int u = 0; u < U; ++u) { s[u][r] = __builtin_amdgcn_exp2f(s[u][r] - off); l[r] += s[u][r]; }
#pragma unroll
            for (int e = 0; e < E; ++e) o[r][e] *= f[r];
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
            float x[E];
            P::open(cur.v[u], x);
#pragma unroll
            for (int r = 0; r < R; ++r)
#pragma unroll
                for (int e = 0; e < E; ++e) o[r][e] = __builtin_fmaf(s[u][r], x[e], o[r][e]);
        }
        cur = nxt;
    }
    // join the groups of the wave, then the waves
#pragma unroll
    for (int r = 0; r < R; ++r) {
#pragma unroll
        for (int w = PP; w < 64; w <<= 1) {
            const float m2 = __shfl_xor(m[r], w, 64), l2 = __shfl_xor(l[r], w, 64), mn = fmaxf(m[r], m2), off = mn == -INFINITY ? 0.f : mn;
            const float f1 = __builtin_amdgcn_exp2f(m[r] - off), f2 = __builtin_amdgcn_exp2f(m2 - off);
            l[r] = l[r] * f1 + l2 * f2;
            m[r] = mn;
#pragma unroll
            for (int e = 0; e < E; ++e) o[r][e] = o[r][e] * f1 + __shfl_xor(o[r][e], w, 64) * f2;
        }
        if (grp == 0) {
            if (p == 0) { sm[wave][r] = m[r]; sl[wave][r] = l[r]; }
#pragma unroll
            for (int e = 0; e < E; ++e) so[wave][r][p * E + e] = o[r][e];
        }
    }
    __syncthreads();
    for (int i = tid; i < R * PP * E; i += 256) {
        const int r = i / (PP * E), c = i - r * (PP * E);
        if (r >= a.G || c >= a.d) continue;
        float mx = fmaxf(fmaxf(sm[0][r], sm[1][r]), fmaxf(sm[2][r], sm[3][r])), off = mx == -INFINITY ? 0.f : mx, ll = 0.f, x = 0.f;
#pragma unroll
        for (int w = 0; w < 4; ++w) {
            const float fw = __builtin_amdgcn_exp2f(sm[w][r] - off);
            ll += sl[w][r] * fw;
            x += so[w][r][c] * fw;
        }
        const int h = hk * a.G + r;
        const long bh = (long)b * a.H + h;
        if (a.nsplit > 1) {
            const long ri = (long)split * a.B * a.H + bh;
            a.part[ri * a.d + c] = x;
            if (c == 0) { a.ml[ri * 2] = mx; a.ml[ri * 2 + 1] = ll; }
            continue;
        }
        const bool none = ll == 0.f;
        x = none ? 0.f : x / ll;
        st1(static_cast<T*>(a.o.p) + b * a.o.batch + h * a.o.head + c, x);
        if (a.o32) a.o32[bh * a.d + c] = x;
        if (c == 0 && a.lse) a.lse[bh] = none ? -INFINITY : (mx + __builtin_amdgcn_logf(ll)) * SEQ_LN2;
    }
#endif
}

// ---------------------------------------------------------------- host side
bool seq_token_takes(const SeqArgs& a) { return a.Nq == 1 && a.G <= 8; }
int seq_token_split(const SeqArgs& a) {
    // two blocks a CU, parts of at least 256 keys. Blocks 512 / 1024 / 2048: 32 x 12 heads over up to 8192 keys 121 + 5 / 120 + 5 / 116 + 8 us (kernel + join),
    // 64 x 4 heads over up to 1500 25 + 4 / 27 + 5 / 28 + 5 us
    const long blocks = (long)a.B * a.Hkv;
    return (int)std::max(1l, std::min<long>(cdiv(512, std::max(blocks, 1l)), a.Nk / 256));
}
template <typename T, int PP, int R>
static void tok_go(const Launch& L, const SeqArgs& a) {
    const dim3 grid((unsigned)a.B * a.Hkv, a.nsplit);
    if (a.table) hipLaunchKernelGGL((seq_token_kernel<T, PP, R, true>), grid, dim3(256), 0, L.stream, a);
    else hipLaunchKernelGGL((seq_token_kernel<T, PP, R, false>), grid, dim3(256), 0, L.stream, a);
    CB_HIP(hipGetLastError());
}
template <typename T, int PP>
static void tok_heads(const Launch& L, const SeqArgs& a) {
    if (a.G == 1) tok_go<T, PP, 1>(L, a);
    else if (a.G == 2) tok_go<T, PP, 2>(L, a);
    else if (a.G <= 4) tok_go<T, PP, 4>(L, a);
    else tok_go<T, PP, 8>(L, a);
}
void seq_token(const Launch& L, const SeqArgs& a) {
    L.count();
    if (L.dry) return;
    const int pieces = a.d * (int)dt_size(a.dt) / 16;
    CB_DT_SWITCH(a.dt, T, {
        if (pieces <= 4) tok_heads<T, 4>(L, a);
        else if (pieces <= 8) tok_heads<T, 8>(L, a);
        else if (pieces <= 16) tok_heads<T, 16>(L, a);
        else if (pieces <= 32) tok_heads<T, 32>(L, a);
        else tok_heads<T, 64>(L, a);
    });
}

}  // namespace cb
