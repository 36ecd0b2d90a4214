// cb_seq_short.hip — forward and dQ of the attention of cb_seq.h for up to SEQ_SHORT keys: image tokens that read a prompt.
//
// All keys and values of one (sample, head) stay in LDS, and the scores of a row over all of them in registers: the softmax needs no running
// maximum, and the row sums of the backward pass come from the probabilities in fp32 on the spot (exact; neither output is read). After K and V
// have arrived once, the waves of a block run by themselves, each over blocks of 16 rows, with the rows of the next block in flight: bound by
// reading Q (and dO) and writing O (dQ) and by what a turn of 16 rows takes. Measured on 64 heads, 4096 x 77, d 40, bf16 (forward / dQ): 22 / 25 us, vector
// units 51 / 48 % of the time, 2 waves a SIMD.
#include "cb_seq.h"
#include <algorithm>

namespace cb {

// keys as the kernels below hold them: NT tiles resident
template <typename T, int DT, int NT> struct SeqShort {
    using G = SeqGeo<T, DT>;
    static constexpr int PAD = NT * G::TK + 16;
    static int lds(int D, bool bias) { return 2 * NT * G::IMG + (bias ? (2 * (D + PAD) + 1) * 4 : 0); }
};

// BWD: dQ (and D), else the forward pass
template <typename T, int DT, int NT, bool BIAS, bool BWD>
__global__ __launch_bounds__(256) void seq_short_kernel(const SeqArgs a, const int nqb, const int turns) {
#ifdef __HIP_DEVICE_COMPILE__      // the host pass needs the launch stub alone
    using G = SeqGeo<T, DT>;
    constexpr int TK = G::TK, KT = G::KT, KS = G::KS, PAD = SeqShort<T, DT, NT>::PAD;
    extern __shared__ __attribute__((aligned(16))) char lds_seq[];
    float* bw = reinterpret_cast<float*>(lds_seq + 2 * NT * G::IMG);
    const int tid = threadIdx.x, lane = tid & 63, l15 = lane & 15, g = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    int rank, b, h;
    if (!seq_item_by_row(a.B, a.H, nqb, blockIdx.x, rank, b, h)) return;
    const int bh = b * a.H + h, hk = h / a.G;
    const int qlen = seq_clamp_len(a.q_len, b, a.Nq), klen = seq_clamp_len(a.kv_len, b, a.Nk), pos0 = seq_pos(a.q_pos, b);
    const T* Q = static_cast<const T*>(a.q.p) + b * a.q.batch + h * a.q.head;
    const T* dO = BWD ? static_cast<const T*>(a.dout.p) + b * a.dout.batch + h * a.dout.head : nullptr;
    const unsigned char* mask = a.mask ? a.mask + b * a.mask_b : nullptr;

    unsigned long long live[NT];
    {
        const T* K = static_cast<const T*>(a.k.p) + b * a.k.batch + hk * a.k.head;
        const T* V = static_cast<const T*>(a.v.p) + b * a.v.batch + hk * a.v.head;
        SeqSlots<T, DT> sk, sv;
        sk.init(a.k.row, a.d, tid);
        sv.init(a.v.row, a.d, tid);
        int byte[NT];
#pragma unroll
        for (int t = 0; t < NT; ++t) byte[t] = seq_mask_byte<TK>(mask, t * TK, klen, lane);
#pragma unroll
        for (int t = 0; t < NT; ++t) {
            live[t] = seq_live<TK>(mask != nullptr, byte[t], t * TK, klen);
            char* dst = lds_seq + 2 * t * G::IMG + wave * 1024;
            sk.dma(K + (long)t * TK * a.k.row, dst, live[t], tid);
            sv.dma(V + (long)t * TK * a.v.row, dst + G::IMG, live[t], tid);
        }
    }
    // this wave's blocks of 16 rows: rb, rb + 4, ...
    int rb = rank * (4 * turns) + wave;
    const int rb1 = min(rank * (4 * turns) + 4 * turns, (a.Nq + 15) / 16);
    SeqFrag<T> qf[KS], df[KS], qn[KS] = {}, dn[KS] = {};
    float lse = 0.f, lsen = 0.f;
    auto load = [&](int r, SeqFrag<T> (&q)[KS], SeqFrag<T> (&d)[KS], float& ls) {
        const int row = 16 * r + l15;
        const bool valid = row < qlen;
#pragma unroll
        for (int s = 0; s < KS; ++s) {
            q[s] = seq_frag_row<T>(Q + (long)row * a.q.row, valid, s, g, a.d);
            if constexpr (BWD) d[s] = seq_frag_row<T>(dO + (long)row * a.dout.row, valid, s, g, a.d);
        }
        if constexpr (BWD) ls = valid ? a.lse[(long)bh * a.Nq + row] : -INFINITY;
    };
    if (rb < rb1) load(rb, qf, df, lse);
    if constexpr (BIAS) seq_bias_fill(bw, a, h, PAD, tid);
    asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
    __syncthreads();
    const float scale2 = a.scale * SEQ_L2E;
    for (; rb < rb1; rb += 4) {
        if (rb + 4 < rb1) load(rb + 4, qn, dn, lsen);
        const int q0 = 16 * rb, row = q0 + l15, p0 = pos0 + q0;
        f32x4 s[NT][1][KT], dp[NT][KT];
        // 16 keys at a time; wave-uniform: none of them visible (nothing is computed for them), all, or some
        auto bits = [&](int t, int kt) { return (unsigned)(live[t] >> (16 * kt)) & 0xffffu; };
#pragma unroll
        for (int t = 0; t < NT; ++t)
#pragma unroll
            for (int kt = 0; kt < KT; ++kt) {
                s[t][0][kt] = (f32x4){0.f, 0.f, 0.f, 0.f}; dp[t][kt] = s[t][0][kt];
                if (!bits(t, kt)) continue;
                const char* Ks = lds_seq + 2 * t * G::IMG;
#pragma unroll
                for (int ks = 0; ks < KS; ++ks) {
                    s[t][0][kt] = seq_mma(seq_frag_lds<T, DT>(Ks, kt, ks, l15, g), qf[ks], s[t][0][kt]);
                    if constexpr (BWD) dp[t][kt] = seq_mma(seq_frag_lds<T, DT>(Ks + G::IMG, kt, ks, l15, g), df[ks], dp[t][kt]);
                }
            }
        // scores in the log2 domain, minus infinity where a key is not visible
        float m = -INFINITY;
#pragma unroll
        for (int t = 0; t < NT; ++t) {
            const int k0 = t * TK, hi = k0 + TK - 1 - p0, lo = k0 - p0 - 15;
            const bool far = !BIAS || hi <= -a.D || lo >= a.D;        // one bias for the whole tile
            const float cb = !BIAS ? 0.f : hi <= -a.D ? bw[PAD] : lo >= a.D ? bw[2 * a.D + PAD] : 0.f;
            const float* w = bw + (far ? 0 : k0 + 4 * g - p0 - l15 + a.D + PAD);
#pragma unroll
            for (int kt = 0; kt < KT; ++kt) {
                const unsigned bt = bits(t, kt);
                if (!bt) continue;
                f32x4& x = s[t][0][kt];
                if (far) {
#pragma unroll
                    for (int r = 0; r < 4; ++r) x[r] = __builtin_fmaf(x[r], scale2, cb);
                } else {
#pragma unroll
                    for (int r = 0; r < 4; ++r) x[r] = __builtin_fmaf(x[r], scale2, w[16 * kt + r]);
                }
                if (bt != 0xffffu || (a.causal && k0 + 16 * kt + 15 > p0)) {
                    seq_pin(x);
                    const unsigned nib = bt >> (4 * g);
#pragma unroll
                    for (int r = 0; r < 4; ++r) {
                        const bool ok = ((nib >> r) & 1) && (!a.causal || k0 + 16 * kt + 4 * g + r <= p0 + l15);
                        x[r] = ok ? x[r] : -INFINITY;
                    }
                }
                if constexpr (!BWD) m = fmaxf(m, fmaxf(fmaxf(x[0], x[1]), fmaxf(x[2], x[3])));
            }
        }
        f32x4 o[1][G::DA];
#pragma unroll
        for (int t = 0; t < G::DA; ++t) o[0][t] = (f32x4){0.f, 0.f, 0.f, 0.f};
        // The rows that were fetched for the next turn are waited for before this turn's results are stored: stores count as outstanding memory
        // operations too, and a wait behind them would last until they are done (measured: forward 30 us with it, 28 without, 64 heads, 4096 x 77, before the
        // accumulators lay beside the vector registers)
        auto next = [&]() {
#pragma unroll
            for (int s2 = 0; s2 < KS; ++s2) {
                seq_arrived(qn[s2]);
                qf[s2] = qn[s2];
                if constexpr (BWD) { seq_arrived(dn[s2]); df[s2] = dn[s2]; }
            }
            if constexpr (BWD) { asm volatile("" : "+v"(lsen)); lse = lsen; }
        };
        const long ri = (long)bh * a.Nq + row;
        if constexpr (!BWD) {
            float l = 0.f;
            m = seq_group_max(m);
            const float off = m == -INFINITY ? 0.f : m;
#pragma unroll
            for (int t = 0; t < NT; ++t) {
#pragma unroll
                for (int kt = 0; kt < KT; ++kt) {
                    if (!bits(t, kt)) continue;
                    f32x4& x = s[t][0][kt];
#pragma unroll
                    for (int r = 0; r < 4; ++r) x[r] = __builtin_amdgcn_exp2f(x[r] - off);
                    l += (x[0] + x[1]) + (x[2] + x[3]);
                }
                if (live[t]) seq_tmul<T, DT, 1>(o, lds_seq + (2 * t + 1) * G::IMG, s[t], l15, g);
            }
            l = seq_group_sum(l);
            if (row >= qlen) l = 0.f;
            const bool none = l == 0.f;
            const float inv = none ? 0.f : 1.f / l;
            next();
            if (row < a.Nq) {
                T* O = static_cast<T*>(a.o.p) + b * a.o.batch + h * a.o.head + (long)row * a.o.row;
                seq_row4<T, DT>(o[0], a.d, g, [&](int c, float4 v) { st4(O + c, seq_scaled(v, inv, none)); });
                if (g == 0 && a.lse) a.lse[ri] = none ? -INFINITY : (m + __builtin_amdgcn_logf(l)) * SEQ_LN2;
            }
        } else {
            float ls2 = lse == -INFINITY ? INFINITY : lse * SEQ_L2E;             // a row without a visible key: probabilities of zero
            float m2 = ls2, lg = 0.f, D = 0.f;
            const bool big = seq_row_big(ls2);
            if (__any(big)) {                                                    // rows whose statistics are kept in two numbers (seq_row_stats)
                float mx = -INFINITY, l = 0.f;
                auto each = [&](auto&& f) {
#pragma unroll
                    for (int t = 0; t < NT; ++t)
#pragma unroll
                        for (int kt = 0; kt < KT; ++kt) {
                            if (!bits(t, kt)) continue;
                            seq_pin(s[t][0][kt]);
#pragma unroll
                            for (int r = 0; r < 4; ++r) f(s[t][0][kt][r]);
                        }
                };
                each([&](float x) { mx = fmaxf(mx, x); });
                mx = seq_group_max(mx);
                if (big) m2 = mx;
                each([&](float x) { l += __builtin_amdgcn_exp2f(x - m2); });
                l = seq_group_sum(l);
                if (big) lg = __builtin_amdgcn_logf(l);
                ls2 = 0.f;
#pragma unroll
                for (int t = 0; t < NT; ++t)
#pragma unroll
                    for (int kt = 0; kt < KT; ++kt) {
                        if (!bits(t, kt)) continue;
#pragma unroll
                        for (int r = 0; r < 4; ++r) s[t][0][kt][r] = seq_exponent(s[t][0][kt][r], m2, lg);
                    }
            }
#pragma unroll
            for (int t = 0; t < NT; ++t)
#pragma unroll
                for (int kt = 0; kt < KT; ++kt) {
                    if (!bits(t, kt)) continue;
#pragma unroll
                    for (int r = 0; r < 4; ++r) {
                        s[t][0][kt][r] = __builtin_amdgcn_exp2f(s[t][0][kt][r] - ls2);
                        D = __builtin_fmaf(s[t][0][kt][r], dp[t][kt][r], D);
                    }
                }
            const bool none = m2 == INFINITY;
            D = seq_group_sum(D);
            D = none ? 0.f : D;
#pragma unroll
            for (int t = 0; t < NT; ++t) {
#pragma unroll
                for (int kt = 0; kt < KT; ++kt) {
                    if (!bits(t, kt)) continue;
#pragma unroll
                    for (int r = 0; r < 4; ++r) s[t][0][kt][r] *= dp[t][kt][r] - D;
                }
                if (live[t]) seq_tmul<T, DT, 1>(o, lds_seq + 2 * t * G::IMG, s[t], l15, g);
            }
            next();
            if (row < a.Nq) {
                if (g == 0) { a.dvec[ri] = D; a.stat[ri] = m2; a.stat[(long)a.B * a.H * a.Nq + ri] = lg; }
                T* dQ = static_cast<T*>(a.dq.p) + b * a.dq.batch + h * a.dq.head + (long)row * a.dq.row;
                seq_row4<T, DT>(o[0], a.d, g, [&](int c, float4 v) { st4(dQ + c, seq_scaled(v, a.scale, none)); });
            }
        }
    }
#endif
}

// ---------------------------------------------------------------- host side
// (fp32 heads beyond 128: 128 keys and the bias do not fit LDS)
template <typename T, int DT> constexpr int SHORT_KEYS = sizeof(T) == 4 && DT > 8 ? 64 : SEQ_SHORT;
bool seq_short_takes(const SeqArgs& a) { return a.Nk > 0 && a.Nk <= (a.dt == DT_F32 && a.d > 128 ? SHORT_KEYS<float, 10> : SEQ_SHORT); }
template <typename T, int DT, int NT, bool BWD>
static void short_go(const Launch& L, const SeqArgs& a) {
    // blocks of 16 rows a wave: as many as leave 2 blocks (of 4 waves) a CU, at most 8. Forward / whole backward call, us, by turns: 64 heads, 4096 x 77, d 40,
    // bf16 2: 21 / 57, 4: 19 / 55, 8: 21 / 54, 16: 32 / 66; fp32 2: 59 / 195, 4: 54 / 189, 8: 51 / 187, 16: 63 / 199; 32 heads (2 blocks a CU at 4) bf16
    // 2: 12.2 / 39.5, 4: 12.6 / 37.8, 8: 18 / 44
    const long heads = (long)a.B * a.H, rbs = cdiv(a.Nq, 16);
    const int turns = (int)std::max(1l, std::min<long>(8, heads * rbs / (4 * 512)));
    const int nqb = (int)cdiv(rbs, 4 * turns);
    if (!(heads * nqb)) return;
    L.count();
    if (L.dry) return;
    const int lds = SeqShort<T, DT, NT>::lds(a.D, a.table != nullptr);
    const dim3 grid(seq_grid_by_row(a.B, a.H, nqb));
    if (a.table) {
        set_dyn_lds(reinterpret_cast<const void*>(&seq_short_kernel<T, DT, NT, true, BWD>), 160 * 1024);
        hipLaunchKernelGGL((seq_short_kernel<T, DT, NT, true, BWD>), grid, dim3(256), lds, L.stream, a, nqb, turns);
    } else {
        set_dyn_lds(reinterpret_cast<const void*>(&seq_short_kernel<T, DT, NT, false, BWD>), 160 * 1024);
        hipLaunchKernelGGL((seq_short_kernel<T, DT, NT, false, BWD>), grid, dim3(256), lds, L.stream, a, nqb, turns);
    }
    CB_HIP(hipGetLastError());
}
template <typename T, int DT>
static void short_pick(const Launch& L, const SeqArgs& a, bool bwd) {
    constexpr int ONE = 64 / SeqGeo<T, DT>::TK;
    if constexpr (SHORT_KEYS<T, DT> > 64) {
        if (a.Nk > 64) { if (bwd) short_go<T, DT, 2 * ONE, true>(L, a); else short_go<T, DT, 2 * ONE, false>(L, a); return; }
    }
    if (bwd) short_go<T, DT, ONE, true>(L, a); else short_go<T, DT, ONE, false>(L, a);
}
void seq_short(const Launch& L, const SeqArgs& a, bool bwd) {
    CB_DT_SWITCH(a.dt, T, SEQ_DT_SWITCH(a.d, DT, short_pick<T, DT>(L, a, bwd)));
}

}  // namespace cb
