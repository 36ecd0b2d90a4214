// cb_seq_bwd.hip — backward of the attention of cb_seq.h. With p = exp(s - lse) recomputed tile by tile:
//   dP = dO V^T,  D = rowsum(dO * O),  dS = p (dP - D);   dQ = scale dS K,  dK = scale dS^T Q,  dV = P^T dO,  dtable[c] = sum of dS over the
//   pairs whose distance j - i lies in bucket c.
// Two kernels, so that no sum depends on the order of arrival: one block of queries over the keys (dQ, D), one block of keys over the queries of
// all heads that share them (dK, dV, dtable). Both hold the streamed side in LDS row-major and their own side in registers.
//
// Row sums D. Up to SEQ_SHORT keys cb_seq_short.hip stands in for the first kernel and makes them from the probabilities. Longer key axes take D
// from dO and the stored output, whose probabilities were rounded to bf16; that is good for dQ, but not for dtable, which adds dS over whole
// diagonals, where the error of a row sum does not cancel. So with a table the first kernel also adds p dP in fp32 on its way and hands these
// exact sums to the second, which makes dtable.
// (Measured, dtable of 8 x 12 heads, 512 x 512, bf16, against 64 bits: 2e-3 off with D from the output.)
//
// dtable: the distance is constant along the diagonals of a dS tile. Tiles past the table's range add to one number a lane. The others are
// summed over equal qt - kb in registers, then over the 4 rows of a lane by moving row r by r lanes (DPP, what leaves the 16 lanes belongs to
// the next 16 distances), which leaves every lane one distance per 16 x 16 tile; these are added to sums by distance in LDS that every wave has
// for itself, one row index g after the other, so that no two lanes meet: the order of all additions is fixed. A wave's sums are folded by
// bucket at the end of each head. (Measured, this kernel on 8 x 12 heads, 512 x 512, where half of the tiles are near: by columns of a copy
// shifted row by row 54 us, by ds_add_f32 134 us, with a copy of the sums for each g, which costs the third block a CU, 43 us, so 32 us.)
// What bounds them: vector and matrix instructions one after the other, with two waves a SIMD to overlap them (32 rows a wave take over 200 registers).
// 2 x 12 heads, 4096 causal, d 64, bf16, with bias and dtable: dQ 107 - 117 us (vector units 53 % of the time, matrix units 33 %), dK/dV 156 - 171 us (45 %,
// 30 %; LDS 29 %; scores and dP formed in both kernels: 180 GFLOP, 0.68 PFLOP/s). fp32, 16 heads, 1023 x 333, d 80: 37 and 54 us, matrix units 49 and 45 %: one
// wave a SIMD, whose exponentials nothing runs under (6.1 GFLOP for both, 40 us at the rate of a large fp32 product).
#include "cb_seq.h"
#include <algorithm>

namespace cb {

template <typename T, int DT, int QB, bool BIAS> struct SeqDq {
    using G = SeqGeo<T, DT>;
    static constexpr int PAD = G::TK + 16 * QB;
    static int lds(int D) { return 4 * G::IMG + (BIAS ? (int)rup((2 * (D + PAD) + 1) * 4, 16) : 0); }
};

template <typename T, int DT, int QB, bool BIAS>
__global__ __launch_bounds__(256, QB > 1 ? 2 : 1) void seq_dq_kernel(const SeqArgs a, const int nqb) {
#ifdef __HIP_DEVICE_COMPILE__      // the host pass needs the launch stub alone
    using G = SeqGeo<T, DT>;
    constexpr int TK = G::TK, KT = G::KT, KS = G::KS, STAGE = 2 * G::IMG, PAD = SeqDq<T, DT, QB, BIAS>::PAD;
    extern __shared__ __attribute__((aligned(16))) char lds_seq[];
    float* bw = reinterpret_cast<float*>(lds_seq + 2 * STAGE);
    const int tid = threadIdx.x, lane = tid & 63, l15 = lane & 15, g = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    int rank, b, h;
    seq_item(a, blockIdx.x, rank, b, h);
    const int bh = b * a.H + h, hk = h / a.G, qblk = nqb - 1 - rank;
    const int qlen = seq_clamp_len(a.q_len, b, a.Nq), klen = seq_clamp_len(a.kv_len, b, a.Nk), pos0 = seq_pos(a.q_pos, b);
    const int qb0 = qblk * (64 * QB), q0 = qb0 + wave * (16 * QB);
    const T* Q = static_cast<const T*>(a.q.p) + b * a.q.batch + h * a.q.head;
    const T* K = static_cast<const T*>(a.k.p) + b * a.k.batch + hk * a.k.head;
    const T* V = static_cast<const T*>(a.v.p) + b * a.v.batch + hk * a.v.head;
    const T* dO = static_cast<const T*>(a.dout.p) + b * a.dout.batch + h * a.dout.head;
    const unsigned char* mask = a.mask ? a.mask + b * a.mask_b : nullptr;
    int kend = klen;
    if (a.causal) kend = max(0, min(kend, pos0 + min(qb0 + 64 * QB, qlen)));
    if (qb0 >= qlen) kend = 0;
    const int split = blockIdx.y;                                 // part of the key axis
    int t0 = 0, t1 = (kend + TK - 1) / TK;
    if (a.ksplit > 1) {
        const int per = (t1 + a.ksplit - 1) / a.ksplit;
        t0 = min(split * per, t1); t1 = min(t0 + per, t1);
    }

    SeqFrag<T> qf[QB][KS], df[QB][KS];
    float lse2[QB], dsum[QB], own[QB];                            // own: the sum of p dP as this block sees it
#pragma unroll
    for (int qb = 0; qb < QB; ++qb) {
        const int row = q0 + 16 * qb + l15;
        const bool valid = row < qlen;
        const long ri = (long)bh * a.Nq + row;
        // a row without a visible key has lse = -inf: with +inf in its place its probabilities are zero
        float ls = valid ? a.lse[ri] : -INFINITY;
        lse2[qb] = ls == -INFINITY ? INFINITY : ls * SEQ_L2E;
        const T* O = static_cast<const T*>(a.o.p) + b * a.o.batch + h * a.o.head + (long)row * a.o.row;
        const float* O32 = a.o32 ? a.o32 + (((long)b * a.Nq + row) * a.H + h) * a.d : nullptr;
        float ds = 0.f;
#pragma unroll
        for (int s = 0; s < KS; ++s) {
            qf[qb][s] = seq_frag_row<T>(Q + (long)row * a.q.row, valid, s, g, a.d);
            df[qb][s] = seq_frag_row<T>(dO + (long)row * a.dout.row, valid, s, g, a.d);
            float x[8], y[8];
            if constexpr (G::ES == 2) {
#pragma unroll
                for (int e = 0; e < 8; ++e) x[e] = (float)df[qb][s].v[e];
                if (O32) {
                    const int c = 32 * s + 8 * g;
                    const bool in = valid && c < a.d;
                    const float4 y0 = in ? ld4(O32 + c) : make_float4(0.f, 0.f, 0.f, 0.f), y1 = in ? ld4(O32 + c + 4) : y0;
                    y[0] = y0.x; y[1] = y0.y; y[2] = y0.z; y[3] = y0.w; y[4] = y1.x; y[5] = y1.y; y[6] = y1.z; y[7] = y1.w;
                } else {
                    const SeqFrag<T> f = seq_frag_row<T>(O, valid, s, g, a.d);
#pragma unroll
                    for (int e = 0; e < 8; ++e) y[e] = (float)f.v[e];
                }
            } else {
                const SeqFrag<T> f = seq_frag_row<T>(O, valid, s, g, a.d);
#pragma unroll
                for (int e = 0; e < 4; ++e) { x[e] = df[qb][s].v[e]; y[e] = f.v[e]; }
            }
#pragma unroll
            for (int e = 0; e < G::EP; ++e) ds = __builtin_fmaf(x[e], y[e], ds);
        }
        dsum[qb] = seq_group_sum(ds);
        own[qb] = 0.f;
    }
    float lg[QB];
    bool rare = false;                                            // some row of the wave has its statistics in two numbers
#pragma unroll
    for (int qb = 0; qb < QB; ++qb) {
        lg[qb] = 0.f;
        const bool big = seq_row_big(lse2[qb]);
        if (__any(big)) {
            float m, l;
            seq_row_stats<T, KS, BIAS>(a, K, mask, kend, h, pos0 + q0 + 16 * qb, qf[qb], l15, g, m, l);
            if (big) { lse2[qb] = m; lg[qb] = l; }
            rare = true;
        }
    }
    const float scale2 = a.scale * SEQ_L2E;
    f32x4 acc[QB][G::DA];
#pragma unroll
    for (int qb = 0; qb < QB; ++qb)
#pragma unroll
        for (int t = 0; t < G::DA; ++t) acc[qb][t] = (f32x4){0.f, 0.f, 0.f, 0.f};
    SeqSlots<T, DT> sk, sv;
    sk.init(a.k.row, a.d, tid);
    sv.init(a.v.row, a.d, tid);
    if constexpr (BIAS) seq_bias_fill(bw, a, h, PAD, tid);
    const int wbase = wave * 1024;
    auto stage = [&](int t, unsigned long long live) {
        char* dst = lds_seq + (t & 1) * STAGE + wbase;
        sk.dma(K + (long)t * TK * a.k.row, dst, live, tid);
        sv.dma(V + (long)t * TK * a.v.row, dst + G::IMG, live, tid);
    };
    unsigned long long live = 0, next = 0;
    int byte = 0;
    if (t0 < t1) {
        next = seq_live<TK>(mask, seq_mask_byte<TK>(mask, t0 * TK, klen, lane), t0 * TK, klen);
        stage(t0, next);
        byte = seq_mask_byte<TK>(mask, (t0 + 1) * TK, klen, lane);
    }
#pragma unroll
    for (int qb = 0; qb < QB; ++qb) {
        asm volatile("" : "+v"(lse2[qb]), "+v"(dsum[qb]));
#pragma unroll
        for (int s = 0; s < KS; ++s) { seq_arrived(qf[qb][s]); seq_arrived(df[qb][s]); }
    }
    for (int t = t0; t < t1; ++t) {
        asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
        __builtin_amdgcn_s_barrier();
        asm volatile("" ::: "memory");
        live = next;
        if (t + 1 < t1) {
            next = seq_live<TK>(mask, byte, (t + 1) * TK, klen);
            byte = seq_mask_byte<TK>(mask, (t + 2) * TK, klen, lane);
            stage(t + 1, next);
        }
        if (live == 0) continue;
        const char* Ks = lds_seq + (t & 1) * STAGE;
        const char* Vs = Ks + G::IMG;
        const int k0 = t * TK, p0 = pos0 + q0;
        f32x4 s[QB][KT], dp[QB][KT];
#pragma unroll
        for (int qb = 0; qb < QB; ++qb)
#pragma unroll
            for (int kt = 0; kt < KT; ++kt) { s[qb][kt] = (f32x4){0.f, 0.f, 0.f, 0.f}; dp[qb][kt] = s[qb][kt]; }
#pragma unroll
        for (int ks = 0; ks < KS; ++ks)
#pragma unroll
            for (int kt = 0; kt < KT; ++kt) {
                const SeqFrag<T> kf = seq_frag_lds<T, DT>(Ks, kt, ks, l15, g);
                const SeqFrag<T> vf = seq_frag_lds<T, DT>(Vs, kt, ks, l15, g);
#pragma unroll
                for (int qb = 0; qb < QB; ++qb) {
                    s[qb][kt] = seq_mma(kf, qf[qb][ks], s[qb][kt]);
                    dp[qb][kt] = seq_mma(vf, df[qb][ks], dp[qb][kt]);
                }
            }
        float cb = 0.f, sc = scale2;
        if constexpr (BIAS) {
            const int hi = k0 + TK - 1 - p0, lo = k0 - p0 - (16 * QB - 1);
            if (hi <= -a.D) cb = bw[PAD];
            else if (lo >= a.D) cb = bw[2 * a.D + PAD];
            else {
                const float* w = bw + (k0 + 4 * g - p0 - l15 + a.D + PAD);
                sc = 1.f;
#pragma unroll
                for (int qb = 0; qb < QB; ++qb)
#pragma unroll
                    for (int kt = 0; kt < KT; ++kt)
#pragma unroll
                        for (int r = 0; r < 4; ++r) s[qb][kt][r] = __builtin_fmaf(s[qb][kt][r], scale2, w[16 * kt + r - 16 * qb]);
            }
        }
        if (rare) {
#pragma unroll
            for (int qb = 0; qb < QB; ++qb)
#pragma unroll
                for (int kt = 0; kt < KT; ++kt) {
                    seq_pin(s[qb][kt]);
#pragma unroll
                    for (int r = 0; r < 4; ++r) s[qb][kt][r] = seq_exponent(__builtin_fmaf(s[qb][kt][r], sc, cb), lse2[qb], lg[qb]);
                }
            sc = 1.f;
        }
#pragma unroll
        for (int qb = 0; qb < QB; ++qb) {
            const float off = rare ? 0.f : cb - lse2[qb];
#pragma unroll
            for (int kt = 0; kt < KT; ++kt)
#pragma unroll
                for (int r = 0; r < 4; ++r) s[qb][kt][r] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[qb][kt][r], sc, off));
        }
        // zero what is not visible
        if (live != SEQ_ALL<TK>) {
#pragma unroll
            for (int kt = 0; kt < KT; ++kt) {
#pragma unroll
                for (int qb = 0; qb < QB; ++qb) seq_pin(s[qb][kt]);
                const int nib = (int)(unsigned)(live >> (16 * kt + 4 * g));
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    const bool seen = (nib >> r) & 1;
#pragma unroll
                    for (int qb = 0; qb < QB; ++qb) s[qb][kt][r] = seen ? s[qb][kt][r] : 0.f;
                }
            }
        }
        if (a.causal && k0 + TK - 1 > p0) {
#pragma unroll
            for (int qb = 0; qb < QB; ++qb)
#pragma unroll
                for (int kt = 0; kt < KT; ++kt) {
                    seq_pin(s[qb][kt]);
#pragma unroll
                    for (int r = 0; r < 4; ++r) s[qb][kt][r] = k0 + 16 * kt + 4 * g + r <= p0 + 16 * qb + l15 ? s[qb][kt][r] : 0.f;
                }
        }
        if constexpr (BIAS) {
#pragma unroll
            for (int qb = 0; qb < QB; ++qb)
#pragma unroll
                for (int kt = 0; kt < KT; ++kt)
#pragma unroll
                    for (int r = 0; r < 4; ++r) own[qb] = __builtin_fmaf(s[qb][kt][r], dp[qb][kt][r], own[qb]);
        }
#pragma unroll
        for (int qb = 0; qb < QB; ++qb)
#pragma unroll
            for (int kt = 0; kt < KT; ++kt)
#pragma unroll
                for (int r = 0; r < 4; ++r) s[qb][kt][r] *= dp[qb][kt][r] - dsum[qb];
        seq_tmul<T, DT, QB>(acc, Ks, s, l15, g);
    }
#pragma unroll
    for (int qb = 0; qb < QB; ++qb) {
        const int row = q0 + 16 * qb + l15;
        // with a table: the exact sum over this part of the keys; else the one from the output
        const bool none = lse2[qb] == INFINITY;
        const float sum = BIAS ? seq_group_sum(own[qb]) : split == 0 ? dsum[qb] : 0.f, D = none ? 0.f : sum;
        if (row >= a.Nq) continue;
        if (g == 0) {
            const long ri = (long)bh * a.Nq + row, n = (long)a.B * a.H * a.Nq;
            a.dvec[split * n + ri] = D;
            if (split == 0) { a.stat[ri] = lse2[qb]; a.stat[n + ri] = lg[qb]; }
        }
        if (a.ksplit > 1) {
            float* P = a.partq + (((long)split * a.B * a.H + bh) * a.Nq + row) * a.d;
            seq_row4<T, DT>(acc[qb], a.d, g, [&](int c, float4 v) { st4(P + c, seq_scaled(v, a.scale, none)); });
            continue;
        }
        T* dQ = static_cast<T*>(a.dq.p) + b * a.dq.batch + h * a.dq.head + (long)row * a.dq.row;
        seq_row4<T, DT>(acc[qb], a.d, g, [&](int c, float4 v) { st4(dQ + c, seq_scaled(v, a.scale, none)); });
    }
#endif
}

// dtable[c][h] = sum of the parts of all samples and key blocks; one wave a (bucket, head), 64-bit sums
__global__ __launch_bounds__(64) void seq_dtable_kernel(const SeqArgs a, const int n) {
    const int c = blockIdx.x, h = blockIdx.y, lane = threadIdx.x;
    double x = 0.0;
    for (int i = lane; i < a.B * n; i += 64) {
        const int b = i / n, y = i - b * n;
        x += (double)a.tpart[(((long)b * a.H + h) * n + y) * a.nb + c];
    }
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) x += __shfl_xor(x, o, 64);
    if (lane == 0) a.dtable[(long)c * a.H + h] = (float)x;
}

// v moved between the lanes of each 16 (0 where a lane has no source)
template <int CTRL> __device__ __forceinline__ float dpp0(float v) {
    return __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), CTRL, 0xf, 0xf, true));
}
template <typename T, int DT, int KB, bool BIAS, bool TAB> struct SeqDkv {
    using G = SeqGeo<T, DT>;
    static constexpr int PAD = G::TK + 16 * KB + 16, NE = KB + G::KT - 1;
    static int lds(int D) {
        const int w = 2 * (D + PAD) + 1;
        return 4 * G::IMG + (8 * G::TK + 4) * 4 + (BIAS ? (int)rup(w * 4, 16) : 0) + (TAB ? 4 * w * 4 : 0);
    }
};

template <typename T, int DT, int KB, bool BIAS, bool TAB>
__global__ __launch_bounds__(256, KB > 1 ? 2 : 1) void seq_dkv_kernel(const SeqArgs a, const int nkb) {
#ifdef __HIP_DEVICE_COMPILE__      // the host pass needs the launch stub alone
    using G = SeqGeo<T, DT>;
    using S = SeqDkv<T, DT, KB, BIAS, TAB>;
    constexpr int TQ = G::TK, QT = G::KT, KS = G::KS, STAGE = 2 * G::IMG, PAD = S::PAD, NE = S::NE;
    extern __shared__ __attribute__((aligned(16))) char lds_seq[];
    const int W = 2 * (a.D + PAD) + 1;
    // [2 stages][lse, D, m, log2 l][TQ], [2 stages] whether some row of the tile has its statistics in two numbers: lse is 0 then, else m and log2 l unused
    float* rows = reinterpret_cast<float*>(lds_seq + 2 * STAGE);
    int* two = reinterpret_cast<int*>(rows + 8 * TQ);
    float* bw = rows + 8 * TQ + 4;
    float* hist = bw + ((W + 3) & ~3);                                // [4 waves][W]
    const int tid = threadIdx.x, lane = tid & 63, l15 = lane & 15, g = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int kblk = blockIdx.x / (a.B * a.Hkv), bk = blockIdx.x - kblk * (a.B * a.Hkv), b = bk / a.Hkv, hk = bk - b * a.Hkv;   // causal: the long ones first
    const int split = blockIdx.y;
    const int qlen = seq_clamp_len(a.q_len, b, a.Nq), klen = seq_clamp_len(a.kv_len, b, a.Nk), pos0 = seq_pos(a.q_pos, b);
    const int kb0 = kblk * (64 * KB), k0 = kb0 + wave * (16 * KB);
    const T* K = static_cast<const T*>(a.k.p) + b * a.k.batch + hk * a.k.head;
    const T* V = static_cast<const T*>(a.v.p) + b * a.v.batch + hk * a.v.head;
    const unsigned char* mask = a.mask ? a.mask + b * a.mask_b : nullptr;

    SeqFrag<T> kf[KB][KS], vf[KB][KS];
    bool seen[KB];
#pragma unroll
    for (int kb = 0; kb < KB; ++kb) {
        const int key = k0 + 16 * kb + l15;
        seen[kb] = key < klen && (!mask || mask[key] != 0);
#pragma unroll
        for (int s = 0; s < KS; ++s) {
            kf[kb][s] = seq_frag_row<T>(K + (long)key * a.k.row, seen[kb], s, g, a.d);
            vf[kb][s] = seq_frag_row<T>(V + (long)key * a.v.row, seen[kb], s, g, a.d);
        }
    }
    // steps: the query tiles that can see this block's keys, head after head of those that share them
    const int tq0 = a.causal ? max(0, kb0 - pos0) / TQ : 0;
    const int n1 = kb0 < klen ? max(0, (qlen + TQ - 1) / TQ - tq0) : 0;
    int u0 = 0, u1 = n1 * a.G;
    if (a.nsplit > 1) {
        const int per = (u1 + a.nsplit - 1) / a.nsplit;
        u0 = min(split * per, u1); u1 = min(u0 + per, u1);
    }
    f32x4 dk[KB][G::DA], dv[KB][G::DA];
#pragma unroll
    for (int kb = 0; kb < KB; ++kb)
#pragma unroll
        for (int t = 0; t < G::DA; ++t) { dk[kb][t] = (f32x4){0.f, 0.f, 0.f, 0.f}; dv[kb][t] = dk[kb][t]; }
    SeqSlots<T, DT> sq, sd;
    sq.init(a.q.row, a.d, tid);
    sd.init(a.dout.row, a.d, tid);
    const float scale2 = a.scale * SEQ_L2E;
    const int wbase = wave * 1024;
    float ls = 0.f, dd = 0.f;
    // the step that is fetched next: head and query tile
    int hn = hk * a.G, tn = tq0;
    if (u0 < u1) { hn += u0 / n1; tn += u0 % n1; }
    auto advance = [&]() { if (++tn == tq0 + n1) { tn = tq0; ++hn; } };
    // per-row numbers of a tile: fetched ahead of its DMA and not looked at before the end of the step, when they are written to LDS
    auto fetch = [&]() {
        const int row = tn * TQ + tid;
        ls = INFINITY; dd = 0.f;                                  // (a row without a visible key: probabilities of zero)
        if (tid < TQ && row < qlen) {
            const long ri = ((long)b * a.H + hn) * a.Nq + row;
            ls = a.stat[ri];
            dd = a.dvec[ri];
            for (int s = 1; s < a.ksplit; ++s) dd += a.dvec[(long)s * a.B * a.H * a.Nq + ri];
        }
    };
    auto stage = [&](int u) {
        const int r0 = tn * TQ;
        char* dst = lds_seq + (u & 1) * STAGE + wbase;
        const unsigned long long live = seq_live<TQ>(false, 0, r0, qlen);
        sq.dma(static_cast<const T*>(a.q.p) + b * a.q.batch + hn * a.q.head + (long)r0 * a.q.row, dst, live, tid);
        sd.dma(static_cast<const T*>(a.dout.p) + b * a.dout.batch + hn * a.dout.head + (long)r0 * a.dout.row, dst + G::IMG, live, tid);
    };
    auto put = [&](int u) {
        if (tid < TQ) {                                           // (one wave)
            float* w = rows + (u & 1) * 4 * TQ;
            const bool any = __any(seq_row_big(ls));
            if (any) {
                const int row = tn * TQ + tid;
                w[2 * TQ + tid] = ls;
                w[3 * TQ + tid] = row < qlen ? a.stat[((long)(a.B + b) * a.H + hn) * a.Nq + row] : 0.f;
                ls = 0.f;
            }
            w[tid] = ls; w[TQ + tid] = dd;
            if (tid == 0) two[u & 1] = any;
        }
    };
    int h = hn, q0 = tn * TQ, hcur = -1;
    if (u0 < u1) {
        fetch(); stage(u0);
        if constexpr (BIAS) { seq_bias_fill(bw, a, h, PAD, tid); hcur = h; }
        put(u0);
    }
#pragma unroll
    for (int kb = 0; kb < KB; ++kb)
#pragma unroll
        for (int s = 0; s < KS; ++s) { seq_arrived(kf[kb][s]); seq_arrived(vf[kb][s]); }
    float far_l = 0.f, far_r = 0.f;
    float* hw = hist + wave * W;
    auto clear = [&]() {
        for (int i = lane; i < W; i += 64) hw[i] = 0.f;
        far_l = far_r = 0.f;
    };
    auto out_of = [&](int h) { return a.tpart + ((((long)b * a.H + h) * a.nsplit + split) * nkb + kblk) * a.nb; };
    // the sums by distance of head h, folded over the waves and by bucket (all threads of the block)
    auto fold = [&](int h) {
#pragma unroll
        for (int o = 1; o < 64; o <<= 1) { far_l += __shfl_xor(far_l, o, 64); far_r += __shfl_xor(far_r, o, 64); }
        asm volatile("" ::: "memory");
        if (lane == 0) { hw[0] += far_l; hw[W - 1] += far_r; }
        __syncthreads();
        for (int i = tid; i < W; i += 256) {
            hist[i] = (hist[i] + hist[W + i]) + (hist[2 * W + i] + hist[3 * W + i]);
        }
        __syncthreads();
        float* out = out_of(h);
        for (int c = tid >> 3; c < a.nb; c += 32) {                  // 8 lanes a bucket
            const int lo = a.brange[2 * c], hi = a.brange[2 * c + 1];           // distances + D of the bucket, [lo, hi)
            float x = 0.f;
            if (lo < hi) {
                const int i0 = lo == 0 ? 0 : lo + PAD, i1 = hi == 2 * a.D + 1 ? W : hi + PAD;
                for (int i = i0 + (tid & 7); i < i1; i += 8) x += hist[i];
            }
            x += __shfl_xor(x, 1, 64); x += __shfl_xor(x, 2, 64); x += __shfl_xor(x, 4, 64);
            if ((tid & 7) == 0) out[c] = x;
        }
        __syncthreads();
    };
    if constexpr (TAB) {
        clear();
        const int h0 = hk * a.G, ha = u0 < u1 ? h0 + u0 / n1 : h0 + a.G, hb = u0 < u1 ? h0 + (u1 - 1) / n1 : h0 + a.G;
        for (int x = h0; x < h0 + a.G; ++x)                           // heads of the group that this part of the steps does not reach
            if (x < ha || x > hb) for (int c = tid; c < a.nb; c += 256) out_of(x)[c] = 0.f;
    }
    for (int u = u0; u < u1; ++u) {
        asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
        __builtin_amdgcn_s_barrier();
        asm volatile("" ::: "memory");
        h = hn; q0 = tn * TQ;
        if (BIAS && h != hcur) {
            if (TAB) { fold(hcur); clear(); }
            seq_bias_fill(bw, a, h, PAD, tid);
            hcur = h;
            __syncthreads();
        }
        if (u + 1 < u1) { advance(); fetch(); stage(u + 1); }
        const char* Qs = lds_seq + (u & 1) * STAGE;
        const char* Ds = Qs + G::IMG;
        const float* rw = rows + (u & 1) * 4 * TQ;
        const int pair = two[u & 1];                              // (looked at behind the products, when it is long there)
        const int p0 = pos0 + q0;
        f32x4 s[KB][QT], dp[KB][QT];
#pragma unroll
        for (int kb = 0; kb < KB; ++kb)
#pragma unroll
            for (int qt = 0; qt < QT; ++qt) { s[kb][qt] = (f32x4){0.f, 0.f, 0.f, 0.f}; dp[kb][qt] = s[kb][qt]; }
#pragma unroll
        for (int ks = 0; ks < KS; ++ks)
#pragma unroll
            for (int qt = 0; qt < QT; ++qt) {
                const SeqFrag<T> qf = seq_frag_lds<T, DT>(Qs, qt, ks, l15, g);
                const SeqFrag<T> df = seq_frag_lds<T, DT>(Ds, qt, ks, l15, g);
#pragma unroll
                for (int kb = 0; kb < KB; ++kb) {
                    s[kb][qt] = seq_mma(qf, kf[kb][ks], s[kb][qt]);
                    dp[kb][qt] = seq_mma(df, vf[kb][ks], dp[kb][qt]);
                }
            }
        float cb = 0.f, sc = scale2;
        int side = 0;                                             // -1 / 1: past the table's range on the left / right, 0: by distance
        if constexpr (BIAS) {
            const int hi = k0 + 16 * KB - 1 - p0, lo = k0 - p0 - (TQ - 1);
            if (hi <= -a.D) { cb = bw[PAD]; side = -1; }
            else if (lo >= a.D) { cb = bw[2 * a.D + PAD]; side = 1; }
            else {
                const float* w = bw + (k0 + l15 - p0 - 4 * g + a.D + PAD);
                sc = 1.f;
#pragma unroll
                for (int kb = 0; kb < KB; ++kb)
#pragma unroll
                    for (int qt = 0; qt < QT; ++qt)
#pragma unroll
                        for (int r = 0; r < 4; ++r) s[kb][qt][r] = __builtin_fmaf(s[kb][qt][r], scale2, w[16 * kb - 16 * qt - r]);
            }
        }
        if (__builtin_amdgcn_readfirstlane(pair)) {
#pragma unroll
            for (int qt = 0; qt < QT; ++qt) {
                const f32x4 m = *reinterpret_cast<const f32x4*>(rw + 2 * TQ + 16 * qt + 4 * g), l = *reinterpret_cast<const f32x4*>(rw + 3 * TQ + 16 * qt + 4 * g);
#pragma unroll
                for (int kb = 0; kb < KB; ++kb) {
                    seq_pin(s[kb][qt]);
#pragma unroll
                    for (int r = 0; r < 4; ++r) s[kb][qt][r] = seq_exponent(__builtin_fmaf(s[kb][qt][r], sc, cb), m[r], l[r]);
                }
            }
            sc = 1.f; cb = 0.f;
        }
        const bool full = !a.causal || k0 + 16 * KB - 1 <= p0;
#pragma unroll
        for (int qt = 0; qt < QT; ++qt) {
            const f32x4 lq = *reinterpret_cast<const f32x4*>(rw + 16 * qt + 4 * g), dq = *reinterpret_cast<const f32x4*>(rw + TQ + 16 * qt + 4 * g);
#pragma unroll
            for (int kb = 0; kb < KB; ++kb)
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    const float p = __builtin_amdgcn_exp2f(__builtin_fmaf(s[kb][qt][r], sc, cb - lq[r]));
                    s[kb][qt][r] = p;
                    dp[kb][qt][r] = p * (dp[kb][qt][r] - dq[r]);
                }
        }
        if (!full) {
#pragma unroll
            for (int kb = 0; kb < KB; ++kb)
#pragma unroll
                for (int qt = 0; qt < QT; ++qt) {
                    seq_pin(s[kb][qt]); seq_pin(dp[kb][qt]);
#pragma unroll
                    for (int r = 0; r < 4; ++r)
                        if (k0 + 16 * kb + l15 > p0 + 16 * qt + 4 * g + r) { s[kb][qt][r] = 0.f; dp[kb][qt][r] = 0.f; }
                }
        }
        if constexpr (TAB) {
            // (columns of keys that are not visible hold anything)
#pragma unroll
            for (int kb = 0; kb < KB; ++kb)
                if (!__all(seen[kb])) {
#pragma unroll
                    for (int qt = 0; qt < QT; ++qt) {
                        seq_pin(dp[kb][qt]);
#pragma unroll
                        for (int r = 0; r < 4; ++r) dp[kb][qt][r] = seen[kb] ? dp[kb][qt][r] : 0.f;
                    }
                }
            if (side != 0) {
                float sum = 0.f;
#pragma unroll
                for (int kb = 0; kb < KB; ++kb)
#pragma unroll
                    for (int qt = 0; qt < QT; ++qt) sum += (dp[kb][qt][0] + dp[kb][qt][1]) + (dp[kb][qt][2] + dp[kb][qt][3]);
                if (side < 0) far_l += sum; else far_r += sum;
            } else {
                f32x4 x[NE];                                      // by e = qt - kb + KB - 1
#pragma unroll
                for (int e = 0; e < NE; ++e) {
                    x[e] = (f32x4){0.f, 0.f, 0.f, 0.f};
#pragma unroll
                    for (int kb = 0; kb < KB; ++kb) {
                        const int qt = e - (KB - 1) + kb;
                        if (qt >= 0 && qt < QT) x[e] += dp[kb][qt];
                    }
                }
                float y[NE + 1];
                y[0] = 0.f;
#pragma unroll
                for (int e = 0; e < NE; ++e) {
                    y[e] += x[e][0] + dpp0<0x101>(x[e][1]) + dpp0<0x102>(x[e][2]) + dpp0<0x103>(x[e][3]);          // row_shl: lane l takes lane l + r
                    y[e + 1] = dpp0<0x11F>(x[e][1]) + dpp0<0x11E>(x[e][2]) + dpp0<0x11D>(x[e][3]);                 // row_shr by 16 - r: the lanes below r
                }
                float* hb = hw + (k0 - p0 + l15 - 4 * g + a.D + PAD + 16 * (KB - 1));
                for (int q = 0; q < 4; ++q) {
                    asm volatile("" ::: "memory");                // one wave's LDS accesses execute in order
                    if (g != q) continue;
                    float o[NE + 1];
#pragma unroll
                    for (int e = 0; e <= NE; ++e) o[e] = hb[-16 * e];
#pragma unroll
                    for (int e = 0; e <= NE; ++e) hb[-16 * e] = o[e] + y[e];
                }
                asm volatile("" ::: "memory");
            }
        }
        seq_tmul<T, DT, KB>(dv, Ds, s, l15, g);
        seq_tmul<T, DT, KB>(dk, Qs, dp, l15, g);
        if (u + 1 < u1) put(u + 1);
    }
    if constexpr (TAB) { if (hcur >= 0) fold(hcur); }
#pragma unroll
    for (int kb = 0; kb < KB; ++kb) {
        const int key = k0 + 16 * kb + l15;
        if (key >= a.Nk) continue;
        const float f = seen[kb] ? 1.f : 0.f, fs = seen[kb] ? a.scale : 0.f;
        const bool hid = !seen[kb];
        if (a.nsplit > 1) {
            const long n = (long)a.B * a.Hkv * a.Nk, ri = (long)bk * a.Nk + key;
            float* P = a.part + ((long)split * 2 * n + ri) * a.d;
            seq_row4<T, DT>(dk[kb], a.d, g, [&](int c, float4 v) { st4(P + c, hid ? make_float4(0.f, 0.f, 0.f, 0.f) : make_float4(v.x * fs, v.y * fs, v.z * fs, v.w * fs)); });
            P += n * a.d;
            seq_row4<T, DT>(dv[kb], a.d, g, [&](int c, float4 v) { st4(P + c, hid ? make_float4(0.f, 0.f, 0.f, 0.f) : v); });
            continue;
        }
        T* dK = static_cast<T*>(a.dk.p) + b * a.dk.batch + hk * a.dk.head + (long)key * a.dk.row;
        T* dV = static_cast<T*>(a.dv.p) + b * a.dv.batch + hk * a.dv.head + (long)key * a.dv.row;
        seq_row4<T, DT>(dk[kb], a.d, g, [&](int c, float4 v) { st4(dK + c, hid ? make_float4(0.f, 0.f, 0.f, 0.f) : make_float4(v.x * fs, v.y * fs, v.z * fs, v.w * fs)); });
        seq_row4<T, DT>(dv[kb], a.d, g, [&](int c, float4 v) { st4(dV + c, hid ? make_float4(0.f, 0.f, 0.f, 0.f) : v); });
    }
#endif
}

// gradients from the parts of a split axis, in order: dK and dV ([nsplit][2][B][Hkv][Nk][d]) or dQ ([ksplit][B][H][Nq][d]); one thread per 4 columns
template <typename T>
__global__ __launch_bounds__(256) void seq_sum_kernel(const float* __restrict__ part, const SeqT d0, const SeqT d1, const int nsplit, const int two, const int B, const int H,
                                                      const int N, const int d) {
    const int d4 = d >> 2;
    const long n = (long)B * H * N, rows = two ? 2 * n : n, i = (long)blockIdx.x * 256 + threadIdx.x;
    if (i >= rows * d4) return;
    const long rr = i / d4;
    const int c = (int)(i - rr * d4) * 4;
    const bool second = rr >= n;
    const long ri = second ? rr - n : rr;
    float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
    for (int s = 0; s < nsplit; ++s) {
        const float4 v = ld4(part + (s * rows + rr) * d + c);
        x.x += v.x; x.y += v.y; x.z += v.z; x.w += v.w;
    }
    const long bh = ri / N, row = ri - bh * N, b = bh / H, h = bh - b * H;
    const SeqT& t = second ? d1 : d0;
    st4(static_cast<T*>(t.p) + b * t.batch + h * t.head + row * t.row + c, x);
}

// ---------------------------------------------------------------- host side
SeqBwdPlan seq_bwd_plan(const SeqArgs& a, bool want_dtable) {
    SeqBwdPlan p;
    const bool wide = a.dt == DT_BF16 && a.d <= 64;                  // what the registers hold for 32 rows a wave
    const long bh = (long)a.B * a.H, bk = (long)a.B * a.Hkv;
    // measured, the whole call with a table. dQ with 16 / 32 rows a wave: 384 blocks of 128 queries (8 x 12 heads, 512 x 512) 53.7 / 56.3 us, 600 (10 x 12
    // heads, 600 x 600) 92.5 / 98.0, 768 (2 x 12 heads, 4096 causal) 257 / 247. dK, dV: 384 blocks of 128 keys 53.7 / 56.9 us, 600 92.5 / 100.9, 768 262 / 247
    p.qb = wide && bh * cdiv(a.Nq, 128) >= 768 ? 2 : 1;
    p.kb = wide && bk * cdiv(a.Nk, 128) >= 768 ? 2 : 1;
    p.nqb = (int)cdiv(a.Nq, 64 * p.qb);
    const bool brief = seq_short_takes(a);
    p.nkb = (int)cdiv(a.Nk, 64 * p.kb);
    // few blocks of keys (or queries): the other axis is split into runs of at least 4 tiles. 128 blocks (64 heads, 4096 x 77, d 40), whole call:
    // 99 us unsplit, 55 us in 8 parts
    const long fill = a.dt == DT_BF16 ? 1024 : 512;
    const long kblocks = bk * cdiv(a.Nk, 64 * p.kb), steps = (long)a.G * cdiv(a.Nq, 64);
    p.qsplit = kblocks < 384 && steps >= 8 ? (int)std::min<long>(fill / std::max(kblocks, 1l), steps / 4) : 1;
    const long qblocks = bh * p.nqb, tiles = cdiv(a.Nk, 64);
    p.ksplit = qblocks < 256 && tiles >= 8 && a.Nk > SEQ_SHORT ? (int)std::min<long>(cdiv(512, std::max(qblocks, 1l)), tiles / 4) : 1;
    if (brief) { p.qb = 0; p.ksplit = 1; }                          // cb_seq_short.hip makes dQ and D
    p.dvec = (size_t)rup((long)p.ksplit * a.B * a.H * a.Nq * 4, 256);
    p.stat = (size_t)rup((long)2 * a.B * a.H * a.Nq * 4, 256);
    p.tpart = want_dtable ? (size_t)rup((long)a.B * a.H * p.qsplit * p.nkb * a.nb * 4, 256) : 0;
    p.part = p.qsplit > 1 ? (size_t)rup((long)p.qsplit * 2 * a.B * a.Hkv * a.Nk * a.d * 4, 256) : 0;
    p.partq = p.ksplit > 1 ? (size_t)p.ksplit * a.B * a.H * a.Nq * a.d * 4 : 0;
    p.total = p.dvec + p.stat + p.tpart + p.part + p.partq;
    return p;
}
template <typename T, int DT, int QB, bool BIAS>
static void dq_go(const Launch& L, const SeqArgs& a, int nqb) {
    if (!((long)nqb * a.B)) return;
    L.count();
    if (L.dry) return;
    const int lds = SeqDq<T, DT, QB, BIAS>::lds(a.D);
    set_dyn_lds(reinterpret_cast<const void*>(&seq_dq_kernel<T, DT, QB, BIAS>), 160 * 1024);
    hipLaunchKernelGGL((seq_dq_kernel<T, DT, QB, BIAS>), dim3((unsigned)nqb * a.B * a.H, a.ksplit), dim3(256), lds, L.stream, a, nqb);
    CB_HIP(hipGetLastError());
}
template <typename T, int DT, int KB, bool BIAS, bool TAB>
static void dkv_go(const Launch& L, const SeqArgs& a) {
    const int nkb = (int)cdiv(a.Nk, 64 * KB);
    if (!((long)nkb * a.B)) return;
    L.count();
    if (L.dry) return;
    const int lds = SeqDkv<T, DT, KB, BIAS, TAB>::lds(a.D);
    CB_CHECK(lds <= 160 * 1024, CB_ERR_SHAPE, "seq attention: %d bytes of LDS for head dim %d and max_distance %d", lds, a.d, a.D);
    set_dyn_lds(reinterpret_cast<const void*>(&seq_dkv_kernel<T, DT, KB, BIAS, TAB>), 160 * 1024);
    hipLaunchKernelGGL((seq_dkv_kernel<T, DT, KB, BIAS, TAB>), dim3((unsigned)nkb * a.B * a.Hkv, a.nsplit), dim3(256), lds, L.stream, a, nkb);
    CB_HIP(hipGetLastError());
}
template <typename T, int DT, int QB>
static void dq_kind(const Launch& L, const SeqArgs& a, int nqb) {
    if (a.table) dq_go<T, DT, QB, true>(L, a, nqb);
    else dq_go<T, DT, QB, false>(L, a, nqb);
}
template <typename T, int DT, int KB>
static void dkv_kind(const Launch& L, const SeqArgs& a) {
    if (a.table && a.dtable) dkv_go<T, DT, KB, true, true>(L, a);
    else if (a.table) dkv_go<T, DT, KB, true, false>(L, a);
    else dkv_go<T, DT, KB, false, false>(L, a);
}
template <typename T, int DT>
static void bwd_pick(const Launch& L, const SeqArgs& a, const SeqBwdPlan& p) {
    if constexpr (sizeof(T) == 2 && DT <= 4) {
        if (p.qb == 2) dq_kind<T, DT, 2>(L, a, p.nqb); else if (p.qb == 1) dq_kind<T, DT, 1>(L, a, p.nqb);
        if (p.kb == 2) dkv_kind<T, DT, 2>(L, a); else dkv_kind<T, DT, 1>(L, a);
    } else {
        if (p.qb) dq_kind<T, DT, 1>(L, a, p.nqb);
        dkv_kind<T, DT, 1>(L, a);
    }
}
static void sum_parts(const Launch& L, DType dt, const float* part, const SeqT& d0, const SeqT& d1, int nsplit, int two, int B, int H, int N, int d) {
    const long n = (long)(two ? 2 : 1) * B * H * N * (d / 4);
    if (!n) return;
    L.count();
    if (L.dry) return;
    CB_DT_SWITCH(dt, T, hipLaunchKernelGGL((seq_sum_kernel<T>), dim3(cdiv(n, 256)), dim3(256), 0, L.stream, part, d0, d1, nsplit, two, B, H, N, d));
    CB_HIP(hipGetLastError());
}
void seq_backward(const Launch& L, SeqArgs a, void* ws) {
    const SeqBwdPlan p = seq_bwd_plan(a, a.dtable != nullptr);
    char* w = static_cast<char*>(ws);
    a.dvec = reinterpret_cast<float*>(w); w += p.dvec;
    a.stat = reinterpret_cast<float*>(w); w += p.stat;
    a.tpart = reinterpret_cast<float*>(w); w += p.tpart;
    a.part = reinterpret_cast<float*>(w); w += p.part;
    a.partq = reinterpret_cast<float*>(w);
    a.nsplit = p.qsplit;
    a.ksplit = p.ksplit;
    if (p.qb == 0) seq_short(L, a, true);
    CB_DT_SWITCH(a.dt, T, SEQ_DT_SWITCH(a.d, DT, bwd_pick<T, DT>(L, a, p)));
    if (a.dtable) {
        L.count();
        if (!L.dry) {
            hipLaunchKernelGGL(seq_dtable_kernel, dim3(a.nb, a.H), dim3(64), 0, L.stream, a, p.nkb * p.qsplit);
            CB_HIP(hipGetLastError());
        }
    }
    if (a.ksplit > 1) sum_parts(L, a.dt, a.partq, a.dq, a.dq, a.ksplit, 0, a.B, a.H, a.Nq, a.d);
    if (a.nsplit > 1) sum_parts(L, a.dt, a.part, a.dk, a.dv, a.nsplit, 1, a.B, a.Hkv, a.Nk, a.d);
}

}  // namespace cb
