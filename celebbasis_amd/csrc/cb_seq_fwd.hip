// cb_seq_fwd.hip — forward of the attention of cb_seq.h (lengths, key masks, shared heads, relative position bias).
//
// One pass over the keys with the running maximum and sum of the softmax: S^T = K Q^T, p = exp2(s - m), O^T += V^T P^T, the probabilities
// going from the first product's accumulators into the second's operand inside the lane. A block has 4 waves of 16 QB queries of one (sample,
// head); K and V tiles come by LDS-DMA into a ring of two stages (one wait and one barrier a tile). Bound by scores, exponentials and P V one after the
// other in a wave, with 2 waves a SIMD: 2 x 12 heads, 4096 causal, d 64, bf16 82 - 89 us, vector units 56 % of the time, matrix units 29 %, LDS 23 %;
// 4 x 16 heads on 4, 1024 x 2000, mask, d 128 77 - 89 us, 59 %, 36 %, 27 %.
#include "cb_seq.h"
#include <algorithm>

namespace cb {

template <typename T, int DT, int QB, bool BIAS>
__global__ __launch_bounds__(256, DT > 8 ? 1 : 2) void seq_fwd_kernel(const SeqArgs a, const int nqb) {
#ifdef __HIP_DEVICE_COMPILE__      // the host pass needs the launch stub alone
    using G = SeqGeo<T, DT>;
    constexpr int TK = G::TK, KT = G::KT, KS = G::KS, STAGE = 2 * G::IMG, PAD = TK + 16 * QB;
    extern __shared__ __attribute__((aligned(16))) char lds_seq[];
    float* bw = reinterpret_cast<float*>(lds_seq + 2 * STAGE);
    const int tid = threadIdx.x, lane = tid & 63, l15 = lane & 15, g = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    int rank, b, h;
    seq_item(a, blockIdx.x, rank, b, h);
    const int bh = b * a.H + h, hk = h / a.G, qblk = nqb - 1 - rank;                 // causal: the long rows first
    const int split = blockIdx.y;
    const int qlen = seq_clamp_len(a.q_len, b, a.Nq), klen = seq_clamp_len(a.kv_len, b, a.Nk), pos0 = seq_pos(a.q_pos, b);
    const int qb0 = qblk * (64 * QB), q0 = qb0 + wave * (16 * QB);
    const T* Q = static_cast<const T*>(a.q.p) + b * a.q.batch + h * a.q.head;
    const T* K = static_cast<const T*>(a.k.p) + b * a.k.batch + hk * a.k.head;
    const T* V = static_cast<const T*>(a.v.p) + b * a.v.batch + hk * a.v.head;
    const unsigned char* mask = a.mask ? a.mask + b * a.mask_b : nullptr;

    // keys this block has to look at: up to the sample's length and, causal, the block's last position
    int kend = klen;
    if (a.causal) kend = max(0, min(kend, pos0 + min(qb0 + 64 * QB, qlen)));
    if (qb0 >= qlen) kend = 0;
    int t0 = 0, t1 = (kend + TK - 1) / TK;
    if (a.nsplit > 1) {
        const int per = (t1 + a.nsplit - 1) / a.nsplit;
        t0 = min(split * per, t1); t1 = min(t0 + per, t1);
    }

    SeqFrag<T> qf[QB][KS];
#pragma unroll
    for (int qb = 0; qb < QB; ++qb)
#pragma unroll
        for (int s = 0; s < KS; ++s) {
            const int row = q0 + 16 * qb + l15;
            qf[qb][s] = seq_frag_row<T>(Q + (long)row * a.q.row, row < qlen, s, g, a.d);
        }
    const float scale2 = a.scale * SEQ_L2E;
    f32x4 o[QB][G::DA];
    float m[QB], l[QB];
#pragma unroll
    for (int qb = 0; qb < QB; ++qb) {
        m[qb] = -INFINITY; l[qb] = 0.f;
#pragma unroll
        for (int t = 0; t < G::DA; ++t) o[qb][t] = (f32x4){0.f, 0.f, 0.f, 0.f};
    }
    SeqSlots<T, DT> sk, sv;
    sk.init(a.k.row, a.d, tid);
    sv.init(a.v.row, a.d, tid);
    int far = 0;
    if constexpr (BIAS) {
        seq_bias_fill(bw, a, h, PAD, tid);
        far = seq_bias_far(a, h);
    }
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
    for (int qb = 0; qb < QB; ++qb)
#pragma unroll
        for (int s = 0; s < KS; ++s) seq_arrived(qf[qb][s]);
    for (int t = t0; t < t1; ++t) {
        // tile t has landed for this wave and, behind the barrier, for all; everybody has read the other stage, which is filled next
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
        const int k0 = t * TK;
        f32x4 s[QB][KT];
#pragma unroll
        for (int qb = 0; qb < QB; ++qb)
#pragma unroll
            for (int kt = 0; kt < KT; ++kt) s[qb][kt] = (f32x4){0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int ks = 0; ks < KS; ++ks)
#pragma unroll
            for (int kt = 0; kt < KT; ++kt) {
                const SeqFrag<T> kf = seq_frag_lds<T, DT>(Ks, kt, ks, l15, g);
#pragma unroll
                for (int qb = 0; qb < QB; ++qb) s[qb][kt] = seq_mma(kf, qf[qb][ks], s[qb][kt]);
            }
        // the bias: one number for the whole tile where every distance is past the table's range, else by distance from LDS; s is then in the
        // log2 domain already (sc = 1). (Tiles past the range that come here all the same are moved to where bw holds that number throughout.)
        const int p0 = pos0 + q0;
        float cb = 0.f, sc = scale2;
        if constexpr (BIAS) {
            const int hi = k0 + TK - 1 - p0, lo = k0 - p0 - (16 * QB - 1);
            if (hi <= -far) cb = bw[PAD];
            else if (lo >= far) cb = bw[2 * a.D + PAD];
            else {
                const int at = min(max(k0 - p0, -(a.D + TK - 1)), a.D + 16 * QB - 1);
                const float* w = bw + (at + 4 * g - l15 + a.D + PAD);
                sc = 1.f;
#pragma unroll
                for (int qb = 0; qb < QB; ++qb)
#pragma unroll
                    for (int kt = 0; kt < KT; ++kt)
#pragma unroll
                        for (int r = 0; r < 4; ++r) s[qb][kt][r] = __builtin_fmaf(s[qb][kt][r], scale2, w[16 * kt + r - 16 * qb]);
            }
        }
        if (live != SEQ_ALL<TK>) {                   // keys that the length or the mask hides
#pragma unroll
            for (int kt = 0; kt < KT; ++kt) {
#pragma unroll
                for (int qb = 0; qb < QB; ++qb) seq_pin(s[qb][kt]);
                const int nib = (int)~(unsigned)(live >> (16 * kt + 4 * g));
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    const float hid = __int_as_float(((nib << (31 - r)) >> 31) & 0xFF800000);        // 0 or -inf
#pragma unroll
                    for (int qb = 0; qb < QB; ++qb) s[qb][kt][r] += hid;
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
                    for (int r = 0; r < 4; ++r) s[qb][kt][r] = k0 + 16 * kt + 4 * g + r <= p0 + 16 * qb + l15 ? s[qb][kt][r] : -INFINITY;
                }
        }
        // The exponent's reference m follows the running maximum only where a lane is more than 8 (2^8) above it: p stays below 2^8, which costs
        // nothing in fp32 sums or in bf16's relative rounding, and most tiles need neither the maximum over the lanes of a row nor a rescaling.
        // (m is the same in the 4 lanes of a row.) The sum l stays apart by lane until the end.
#pragma unroll
        for (int qb = 0; qb < QB; ++qb) {
            float mx = -INFINITY;
#pragma unroll
            for (int kt = 0; kt < KT; ++kt)
#pragma unroll
                for (int r = 0; r < 4; ++r) mx = fmaxf(mx, s[qb][kt][r]);
            mx = __builtin_fmaf(mx, sc, cb);
            if (__any(mx > m[qb] + 8.f)) {
                const float mnew = fmaxf(m[qb], seq_group_max(mx));
                const float alpha = mnew == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(m[qb] - mnew);
#pragma unroll
                for (int t2 = 0; t2 < G::DA; ++t2) o[qb][t2] *= alpha;
                l[qb] *= alpha;
                m[qb] = mnew;
            }
        }
#pragma unroll
        for (int qb = 0; qb < QB; ++qb) {
            const float off = m[qb] == -INFINITY ? 0.f : cb - m[qb];
#pragma unroll
            for (int kt = 0; kt < KT; ++kt) {
#pragma unroll
                for (int r = 0; r < 4; ++r) s[qb][kt][r] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[qb][kt][r], sc, off));
                l[qb] += (s[qb][kt][0] + s[qb][kt][1]) + (s[qb][kt][2] + s[qb][kt][3]);
            }
        }
        seq_tmul<T, DT, QB>(o, Vs, s, l15, g);
    }
#pragma unroll
    for (int qb = 0; qb < QB; ++qb) {
        const int row = q0 + 16 * qb + l15;
        l[qb] = seq_group_sum(l[qb]);
        if (row >= a.Nq) continue;
        const long ri = (long)bh * a.Nq + row;
        if (row >= qlen) l[qb] = 0.f;            // a row behind the sample's last query sees nothing
        if (a.nsplit > 1) {                      // unnormalised; seq_combine_kernel joins the parts
            float* P = a.part + ((long)split * a.B * a.H * a.Nq + ri) * a.d;
            seq_row4<T, DT>(o[qb], a.d, g, [&](int c, float4 v) { st4(P + c, v); });
            if (g == 0) { float* w = a.ml + ((long)split * a.B * a.H * a.Nq + ri) * 2; w[0] = m[qb]; w[1] = l[qb]; }
            continue;
        }
        const bool none = l[qb] == 0.f;          // nothing visible: zeros
        const float inv = none ? 0.f : 1.f / l[qb];
        T* O = static_cast<T*>(a.o.p) + b * a.o.batch + h * a.o.head + (long)row * a.o.row;
        float* O32 = a.o32 ? a.o32 + (((long)b * a.Nq + row) * a.H + h) * a.d : nullptr;
        seq_row4<T, DT>(o[qb], a.d, g, [&](int c, float4 v) {
            v = seq_scaled(v, inv, none);
            st4(O + c, v);
            if (O32) st4(O32 + c, v);
        });
        if (g == 0 && a.lse) a.lse[ri] = none ? -INFINITY : (m[qb] + __builtin_amdgcn_logf(l[qb])) * SEQ_LN2;
    }
#endif
}

// joins the parts of a split key axis: o = sum_s o_s 2^(m_s - m) / sum_s l_s 2^(m_s - m), s in order. One thread per 4 columns.
template <typename T>
__global__ __launch_bounds__(256) void seq_combine_kernel(const SeqArgs a) {
    const int d4 = a.d >> 2;
    const long i = (long)blockIdx.x * 256 + threadIdx.x, rows = (long)a.B * a.H * a.Nq;
    if (i >= rows * d4) return;
    const long ri = i / d4;
    const int c = (int)(i - ri * d4) * 4;
    float m = -INFINITY;
    for (int s = 0; s < a.nsplit; ++s) m = fmaxf(m, a.ml[(s * rows + ri) * 2]);
    float l = 0.f;
    float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
    for (int s = 0; s < a.nsplit; ++s) {
        const float2 w = *reinterpret_cast<const float2*>(a.ml + (s * rows + ri) * 2);
        if (w.y == 0.f) continue;                // a part without visible keys
        const float f = __builtin_amdgcn_exp2f(w.x - (m == -INFINITY ? 0.f : m));
        const float4 v = ld4(a.part + (s * rows + ri) * a.d + c);
        l = __builtin_fmaf(w.y, f, l);
        o.x = __builtin_fmaf(v.x, f, o.x); o.y = __builtin_fmaf(v.y, f, o.y); o.z = __builtin_fmaf(v.z, f, o.z); o.w = __builtin_fmaf(v.w, f, o.w);
    }
    const bool none = l == 0.f;
    const float inv = none ? 0.f : 1.f / l;
    const long bh = ri / a.Nq, row = ri - bh * a.Nq, b = bh / a.H, h = bh - b * a.H;
    const float4 v = make_float4(o.x * inv, o.y * inv, o.z * inv, o.w * inv);
    st4(static_cast<T*>(a.o.p) + b * a.o.batch + h * a.o.head + row * a.o.row + c, v);
    if (a.o32) st4(a.o32 + ((b * a.Nq + row) * a.H + h) * a.d + c, v);
    if (c == 0 && a.lse) a.lse[ri] = none ? -INFINITY : (m + __builtin_amdgcn_logf(l)) * SEQ_LN2;
}

// ---------------------------------------------------------------- host side
template <typename T, int DT, int QB, bool BIAS>
static void fwd_go(const Launch& L, const SeqArgs& a) {
    using G = SeqGeo<T, DT>;
    const int nqb = (int)cdiv(a.Nq, 64 * QB);
    const int lds = 4 * G::IMG + (BIAS ? (int)rup((2 * (a.D + G::TK + 16 * QB) + 1) * 4, 16) : 0);
    L.count();
    if (L.dry) return;
    set_dyn_lds(reinterpret_cast<const void*>(&seq_fwd_kernel<T, DT, QB, BIAS>), 160 * 1024);
    hipLaunchKernelGGL((seq_fwd_kernel<T, DT, QB, BIAS>), dim3((unsigned)nqb * a.B * a.H, a.nsplit), dim3(256), lds, L.stream, a, nqb);
    CB_HIP(hipGetLastError());
}
// 32 queries a wave read every K and V fragment for two products instead of one; where the registers do not hold them (fp32, or heads beyond
// 128) or the grid would not fill the chip, 16
static bool fwd_two(const SeqArgs& a) { return a.dt == DT_BF16 ? a.d <= 128 : a.d <= 32; }
template <typename T, int DT>
static void fwd_pick(const Launch& L, const SeqArgs& a, int qb) {
    if constexpr (sizeof(T) == 2 ? DT <= 8 : DT == 2) {
        if (qb == 2) {
            if (a.table) fwd_go<T, DT, 2, true>(L, a); else fwd_go<T, DT, 2, false>(L, a);
            return;
        }
    }
    if (a.table) fwd_go<T, DT, 1, true>(L, a); else fwd_go<T, DT, 1, false>(L, a);
}
SeqPlan seq_fwd_plan(const SeqArgs& a) {
    SeqPlan p;
    const long bh = (long)a.B * a.H;
    const bool token = seq_token_takes(a);
    // measured, 16 against 32 queries a wave: 384 blocks of 128 queries (8 x 12 heads, 512 x 512, d 64) 17.3 / 18.5 us, 600 (10 x 12 heads, 600 x 600)
    // 28.8 / 27.1 us, 768 (2 x 12 heads, 4096 causal) 85.9 / 77.5 us, 512 (64 heads, 1024 x 2000, d 128) 96.7 / 76.4 us
    p.qb = fwd_two(a) && bh * cdiv(a.Nq, 128) >= 512 ? 2 : 1;
    // fewer blocks than CUs: the key axis is split into runs of at least 4 tiles, joined by seq_combine_kernel (with as many blocks as CUs it does not
    // pay: 16 heads, 1023 x 333, fp32, 25 us whole, 31 us in two parts)
    const long blocks = bh * cdiv(a.Nq, 64 * p.qb);
    const int tiles = (int)cdiv(a.Nk, 64);
    p.nsplit = blocks < 256 && tiles >= 8 ? (int)std::min<long>(cdiv(512, std::max(blocks, 1l)), tiles / 4) : 1;
    if (token) { p.qb = 0; p.nsplit = seq_token_split(a); }
    else if (seq_short_takes(a)) { p.qb = -1; p.nsplit = 1; }
    if (p.nsplit > 1) {
        p.part = (size_t)p.nsplit * a.B * a.H * a.Nq * a.d * 4;
        p.ml = (size_t)p.nsplit * a.B * a.H * a.Nq * 2 * 4;
    }
    p.total = p.part + p.ml;
    return p;
}
void seq_forward(const Launch& L, SeqArgs a, void* ws) {
    const SeqPlan p = seq_fwd_plan(a);
    a.nsplit = p.nsplit;
    a.part = static_cast<float*>(ws);
    a.ml = reinterpret_cast<float*>(static_cast<char*>(ws) + p.part);
    if (p.qb == 0) seq_token(L, a);
    else if (p.qb < 0) seq_short(L, a, false);
    else CB_DT_SWITCH(a.dt, T, SEQ_DT_SWITCH(a.d, DT, fwd_pick<T, DT>(L, a, p.qb)));
    if (a.nsplit > 1) {
        L.count();
        if (L.dry) return;
        CB_DT_SWITCH(a.dt, T, hipLaunchKernelGGL((seq_combine_kernel<T>), dim3(cdiv((long)a.B * a.H * a.Nq * (a.d / 4), 256)), dim3(256), 0, L.stream, a));
        CB_HIP(hipGetLastError());
    }
}

}  // namespace cb
