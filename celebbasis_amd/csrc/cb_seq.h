// cb_seq.h — attention over sequences with lengths, key masks, shared key / value heads and a learned relative position bias: the
// arguments of the kernels (cb_seq_fwd.hip, cb_seq_bwd.hip) and the device pieces that they share.
//
//   visible(i, j) = i < q_len[b]  and  j < kv_len[b]  and  mask[b][j]  and  (not causal or j <= q_pos[b] + i)
//   s_ij = scale * q_i . k_j + table[bucket(j - q_pos[b] - i)][h] ;  o_i = sum_j softmax_j(s_ij) v_j  over the visible keys (none: o_i = 0)
//
// One code for fp32 and bf16. A fragment is 16 bytes of a row (lane (l15, g) of a wave: row l15, piece g of a group of four). bf16: 32 elements
// of the head dim a group, one v_mfma_f32_16x16x32_bf16. fp32: 16 elements a group, four v_mfma_f32_16x16x4_f32 whose k index is g and whose
// i-th call takes element i of the piece — a permutation of the sum over the head dim that both operands share. The accumulator of X Y^T (lane: row 4g + r of X, row l15 of
// Y) is, packed, the second operand of the following product without any movement between lanes.
#pragma once
#include "cb_device.h"
#include <type_traits>

namespace cb {

struct SeqT { void* p = nullptr; long row = 0, head = 0, batch = 0; };       // element strides of one token, one head, one sample

struct SeqArgs {
    DType dt = DT_F32;
    int B = 0, Nq = 0, Nk = 0, H = 0, Hkv = 0, G = 1, d = 0;                 // G = H / Hkv query heads share a key / value head
    SeqT q, k, v, o;
    float scale = 1.f; int causal = 0;
    const int* q_pos = nullptr; const int* q_len = nullptr; const int* kv_len = nullptr;
    const unsigned char* mask = nullptr; long mask_b = 0;
    const float* table = nullptr; const short* bmap = nullptr; const int* brange = nullptr; int D = 0, nb = 0;   // relative bias (relpos handle)
    float* lse = nullptr;                                                     // [B][H][Nq], natural logarithm
    float* o32 = nullptr;                                                     // [B][Nq][H][d]: the unrounded output (bf16, kept for the backward pass)
    // backward
    SeqT dout, dq, dk, dv;
    float* dvec = nullptr;                                                    // [ksplit][B][H][Nq]: row sums D (parts of them where keys are split)
    float* stat = nullptr;                                                    // [2][B][H][Nq]: what the exponents of a row are taken off, and log2 of the sum where that is not in it (seq_row_stats)
    float* dtable = nullptr;                                                  // [nb][H]
    float* tpart = nullptr;                                                   // [B][H][parts of queries][blocks of keys][nb]
    float* part = nullptr; float* ml = nullptr; int nsplit = 1;               // partial results of a split axis (fp32): keys (forward), queries (dK, dV)
    float* partq = nullptr; int ksplit = 1;                                    // ... keys (dQ)
};

struct SeqPlan { int qb = 1, nsplit = 1; size_t part = 0, ml = 0, total = 0; };           // sizes in bytes
struct SeqBwdPlan { int qb = 1, kb = 1, qsplit = 1, ksplit = 1, nqb = 1, nkb = 1; size_t dvec = 0, stat = 0, tpart = 0, part = 0, partq = 0, total = 0; };
SeqPlan seq_fwd_plan(const SeqArgs& a);
SeqBwdPlan seq_bwd_plan(const SeqArgs& a, bool want_dtable);
void seq_forward(const Launch& L, SeqArgs a, void* ws);
bool seq_token_takes(const SeqArgs& a);                 // one new token a sample (cb_seq_token.hip)
int seq_token_split(const SeqArgs& a);
void seq_token(const Launch& L, const SeqArgs& a);
bool seq_short_takes(const SeqArgs& a);                 // up to SEQ_SHORT keys (cb_seq_short.hip): forward and dQ
void seq_short(const Launch& L, const SeqArgs& a, bool bwd);
void seq_backward(const Launch& L, SeqArgs a, void* ws);

constexpr int SEQ_MAX_D = 160, SEQ_MAX_DIST = 1024, SEQ_MAX_BUCKETS = 256;
constexpr int SEQ_SHORT = 128;      // key axes up to here: the backward pass makes its row sums from the probabilities (cb_seq_bwd.hip)

#ifdef __HIPCC__
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef unsigned u32x4s __attribute__((ext_vector_type(4)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) void* lds_vp;
typedef __attribute__((address_space(3))) s16x4* lds_s4;

constexpr float SEQ_L2E = 1.4426950408889634f, SEQ_LN2 = 0.6931471805599453f;
// log2 magnitudes from here on share fp32's 24 bits with what they are added to (a half step of 2^12 is 2^-12): kept apart from it
constexpr float SEQ_BIG = 4096.f;
constexpr int SEQ_OOB = -16;                       // 0xFFFFFFF0 >= num_records: the load returns zeros
template <int TK> constexpr unsigned long long SEQ_ALL = TK == 64 ? ~0ull : 0xFFFFFFFFull;      // every row of a tile is visible
// at the head of a rarely taken, wave-uniform branch: keeps its work on x inside (the compiler would turn it into selects that every tile executes)
__device__ __forceinline__ void seq_pin(f32x4& x) { asm volatile("" : "+v"(x)); }
constexpr int SEQ_POS_LIM = 1 << 29;               // positions are held to +-2^29, so that differences stay inside an int

__device__ __forceinline__ float seq_group_max(float v) { v = fmaxf(v, __shfl_xor(v, 16, 64)); return fmaxf(v, __shfl_xor(v, 32, 64)); }
__device__ __forceinline__ float seq_group_sum(float v) { v += __shfl_xor(v, 16, 64); return v + __shfl_xor(v, 32, 64); }
__device__ __forceinline__ __amdgpu_buffer_rsrc_t seq_srd(const void* p) {
    return __builtin_amdgcn_make_buffer_rsrc(const_cast<void*>(p), 0, 0x7FFFFFFF, 0x00020000);
}

template <typename T> struct SeqFrag;
template <> struct SeqFrag<bf16_t> { bf16x8_t v; };
template <> struct SeqFrag<float> { f32x4 v; };
__device__ __forceinline__ f32x4 seq_mma(const SeqFrag<bf16_t>& a, const SeqFrag<bf16_t>& b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a.v, b.v, c, 0, 0, 0);
}
__device__ __forceinline__ f32x4 seq_mma(const SeqFrag<float>& a, const SeqFrag<float>& b, f32x4 c) {
#pragma unroll
    for (int i = 0; i < 4; ++i) c = __builtin_amdgcn_mfma_f32_16x16x4f32(a.v[i], b.v[i], c, 0, 0, 0);
    return c;
}

// Waits for a fragment's load here. Without it the compiler puts that wait at the fragment's first use, inside the tile loop, where it also waits
// for the LDS-DMA of the next tile that has just been issued. Forward with it / without: 64 heads, 4096 x 77, d 40 21.9 / 23.3 us, 16 heads, 1023 x 333,
// fp32 24.7 / 25.8; whole backward call, 2 x 12 heads, 4096 causal 247 / 249.
template <typename T> __device__ __forceinline__ void seq_arrived(SeqFrag<T>& f) { asm volatile("" : "+v"(f.v)); }
// Geometry of one instantiation. A tile is TK rows in LDS, row-major, P pieces of 16 bytes a row, filled by LDS-DMA in lane-linear slots of
// 256 pieces; piece c of row r lies at place swz(c, r), which puts the 16 rows that a fragment read touches into 16 different bank groups.
template <typename T, int DT> struct SeqGeo {
    static constexpr int ES = sizeof(T), EP = 16 / ES;                        // elements of a piece
    static constexpr int KS = ES == 4 ? DT : (DT + 1) / 2;                    // groups of four pieces of a row
    static constexpr int P = 4 * KS;
    static constexpr int TK = (ES == 4 && DT >= 3) ? 32 : 64;                 // fp32: 64 rows would leave one block a CU
    static constexpr int KT = TK / 16;
    static constexpr int TILE = TK * P * 16, NS = (TILE + 4095) / 4096, IMG = NS * 4096;     // an image takes whole slots
    static constexpr int DA = DT;                                             // 16-wide accumulator tiles across the head dim
    static __device__ __forceinline__ int swz(int c, int r) {
        if constexpr (P % 16 == 0) return c ^ (r & 15);
        else if constexpr (P % 8 == 0) return c ^ ((r >> 1) & 7);
        else return c ^ ((r >> 2) & 3);
    }
};

// per-thread source offsets of a tile's slots (bytes from the tile's first row), and the DMA of one tile: rows whose bit in `live` is
// clear, and elements at or beyond the head dim, are filled with zeros — masked places may hold anything, NaN included
template <typename T, int DT> struct SeqSlots {
    using G = SeqGeo<T, DT>;
    int off[G::NS];
    __device__ __forceinline__ void init(long ld, int d, int tid) {
#pragma unroll
        for (int i = 0; i < G::NS; ++i) {
            const int idx = tid + 256 * i, r = idx / G::P, c = G::swz(idx - r * G::P, r);
            off[i] = (r < G::TK && c * G::EP < d) ? (int)((long)r * ld * G::ES + c * 16) : SEQ_OOB;
        }
    }
    // dst: the tile's image + this wave's 1 KiB piece of a slot
    __device__ __forceinline__ void dma(const T* rows, char* dst, unsigned long long live, int tid) const {
        const __amdgpu_buffer_rsrc_t srd = seq_srd(rows);
        if (live == SEQ_ALL<G::TK>) {
#pragma unroll
            for (int i = 0; i < G::NS; ++i) __builtin_amdgcn_raw_ptr_buffer_load_lds(srd, (lds_vp)(dst + i * 4096), 16, off[i], 0, 0, 0);
        } else {
#pragma unroll
            for (int i = 0; i < G::NS; ++i) {
                const int r = (tid + 256 * i) / G::P;
                __builtin_amdgcn_raw_ptr_buffer_load_lds(srd, (lds_vp)(dst + i * 4096), 16, ((live >> (r & 63)) & 1ull) ? off[i] : SEQ_OOB, 0, 0, 0);
            }
        }
    }
};

// fragment of rows 16 blk + l15, group s of the head dim
template <typename T, int DT>
__device__ __forceinline__ SeqFrag<T> seq_frag_lds(const char* img, int blk, int s, int l15, int g) {
    using G = SeqGeo<T, DT>;
    SeqFrag<T> f;
    f.v = *reinterpret_cast<const decltype(f.v)*>(img + ((blk * 16 + l15) * G::P + G::swz(4 * s + g, l15)) * 16);
    return f;
}
// the same of a row in global memory, zeros where the row is not valid
template <typename T>
__device__ __forceinline__ SeqFrag<T> seq_frag_row(const T* row, bool valid, int s, int g, int d) {
    SeqFrag<T> f;
    const int c = (4 * s + g) * (16 / (int)sizeof(T));
    u32x4s v = {0u, 0u, 0u, 0u};
    if (valid && c < d) v = *reinterpret_cast<const u32x4s*>(row + c);
    f.v = __builtin_bit_cast(decltype(f.v), v);
    return f;
}

// acc[QB][DA] += (tile rows)^T . w: the transposed product of the second half of attention. w[qb][kt] is the accumulator of a product of the
// same tile (lane: tile rows 16 kt + 4g + r, column l15).
//   bf16: w is rounded to bf16 here, by at most 2^-8 of each probability (for O and dV) or dS (for dQ and dK), since the matrix unit takes both
//         operands in one type; sums over w (l, D, dtable) are made of the unrounded fp32 values. Against 64 bits a result's error is then 2.3 - 2.4e-3
//         of its norm, where rounding the result alone leaves 1.7e-3; w in two bf16 parts would leave that alone, at twice the products: forward of
//         2 x 12 heads, 4096 causal 110 us in two parts, 89 as it is. (fp32 rounds nothing.)
//         The A operand (head-dim index l15, k slot 8g + j <-> row 32G + 4g + j, or 32G + 16 + 4g + j - 4) comes from two transposing LDS reads
//         (a 16-lane group reads four rows of 16 elements and gets their columns).
//   fp32: one 8-byte read of row 16 kt + 4g + r at columns 32 tt + 2 l15, + 1 feeds two calls; accumulator 2 tt + e then holds column
//         32 tt + 2 (4g + r) + e, so that a lane owns the 8 consecutive columns 32 tt + 8g .. + 7. An odd last tile is read by itself.
template <typename T, int DT, int QB> using SeqAcc = f32x4[QB][SeqGeo<T, DT>::DA];
template <typename T, int DT, int QB> using SeqScores = f32x4[QB][SeqGeo<T, DT>::KT];
template <typename T, int DT> using SeqRow = f32x4[SeqGeo<T, DT>::DA];
template <typename T, int DT, int QB>
__device__ __forceinline__ void seq_tmul(SeqAcc<T, DT, QB>& acc, const char* img, const SeqScores<T, DT, QB>& w, int l15, int g) {
    using G = SeqGeo<T, DT>;
    if constexpr (G::ES == 2) {
#pragma unroll
        for (int kg = 0; kg < G::KT / 2; ++kg) {
            SeqFrag<bf16_t> b[QB];
#pragma unroll
            for (int qb = 0; qb < QB; ++qb) {
                const f32x4 x = w[qb][2 * kg], y = w[qb][2 * kg + 1];
                b[qb].v = (bf16x8_t){(bf16_t)x[0], (bf16_t)x[1], (bf16_t)x[2], (bf16_t)x[3], (bf16_t)y[0], (bf16_t)y[1], (bf16_t)y[2], (bf16_t)y[3]};
            }
            const int r0 = 4 * g + (l15 >> 2), r1 = r0 + 16;             // row inside the 32-row group
            const int half = (l15 & 3) >> 1, sub = (l15 & 1) * 8;
#pragma unroll
            for (int t = 0; t < G::DA; ++t) {
                const char* p0 = img + ((kg * 32 + r0) * G::P + G::swz(2 * t + half, r0)) * 16 + sub;
                const char* p1 = img + ((kg * 32 + r1) * G::P + G::swz(2 * t + half, r1)) * 16 + sub;
                const s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s4)p0), hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s4)p1);
                SeqFrag<bf16_t> a;
                typedef short s16x8 __attribute__((ext_vector_type(8)));
                a.v = __builtin_bit_cast(bf16x8_t, (s16x8){lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]});
#pragma unroll
                for (int qb = 0; qb < QB; ++qb) acc[qb][t] = seq_mma(a, b[qb], acc[qb][t]);
            }
        }
    } else {
#pragma unroll
        for (int kt = 0; kt < G::KT; ++kt)
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const int row = kt * 16 + 4 * g + r;
#pragma unroll
                for (int tt = 0; tt < DT / 2; ++tt) {
                    const int c = 8 * tt + (l15 >> 1);
                    const f32x2 v = *reinterpret_cast<const f32x2*>(img + (row * G::P + G::swz(c, row)) * 16 + (l15 & 1) * 8);
#pragma unroll
                    for (int qb = 0; qb < QB; ++qb) {
                        acc[qb][2 * tt] = __builtin_amdgcn_mfma_f32_16x16x4f32(v[0], w[qb][kt][r], acc[qb][2 * tt], 0, 0, 0);
                        acc[qb][2 * tt + 1] = __builtin_amdgcn_mfma_f32_16x16x4f32(v[1], w[qb][kt][r], acc[qb][2 * tt + 1], 0, 0, 0);
                    }
                }
                if constexpr (DT % 2) {
                    const int c = 4 * (DT - 1) + (l15 >> 2);
                    const float v = *reinterpret_cast<const float*>(img + (row * G::P + G::swz(c, row)) * 16 + (l15 & 3) * 4);
#pragma unroll
                    for (int qb = 0; qb < QB; ++qb) acc[qb][DT - 1] = __builtin_amdgcn_mfma_f32_16x16x4f32(v, w[qb][kt][r], acc[qb][DT - 1], 0, 0, 0);
                }
            }
    }
}
// one row of such an accumulator (this lane's share) through f(column, value); columns at or beyond d are left out
template <typename T, int DT, typename F>
__device__ __forceinline__ void seq_row4(const SeqRow<T, DT>& acc, int d, int g, F f) {
    using G = SeqGeo<T, DT>;
    constexpr int PAIRS = G::ES == 2 ? 0 : DT / 2;
#pragma unroll
    for (int tt = 0; tt < PAIRS; ++tt) {
        const int c = 32 * tt + 8 * g;
        const f32x4 e = acc[2 * tt], o = acc[2 * tt + 1];
        if (c < d) { f(c, make_float4(e[0], o[0], e[1], o[1])); f(c + 4, make_float4(e[2], o[2], e[3], o[3])); }
    }
#pragma unroll
    for (int t = 2 * PAIRS; t < G::DA; ++t) {
        const int c = 16 * t + 4 * g;
        if (c < d) f(c, make_float4(acc[t][0], acc[t][1], acc[t][2], acc[t][3]));
    }
}

// v times f, or zeros where a row sees nothing: selected, since what it was multiplied with may not be finite
__device__ __forceinline__ float4 seq_scaled(float4 v, float f, bool none) { return none ? make_float4(0.f, 0.f, 0.f, 0.f) : make_float4(v.x * f, v.y * f, v.z * f, v.w * f); }
// the bias of head h at distance rel (within +-D), times log2(e). The entries stay finite in the log2 domain (a table may hold its type's lowest
// value): held to +-1e37; minus infinity and NaN are kept.
__device__ __forceinline__ float seq_bias_of(const SeqArgs& a, int h, int rel) {
    const float b = a.table[(long)a.bmap[rel + a.D] * a.H + h];
    return ((b == -INFINITY || b != b) ? b : fminf(fmaxf(b, -1e37f), 1e37f)) * SEQ_L2E;
}
// the bias of one head by distance in LDS: bw[rel + D + pad]. Distances past D share the outermost bucket.
__device__ __forceinline__ void seq_bias_fill(float* bw, const SeqArgs& a, int h, int pad, int tid) {
    const int n = 2 * (a.D + pad) + 1;
    for (int i = tid; i < n; i += 256) bw[i] = seq_bias_of(a, h, min(max(i - (a.D + pad), -a.D), a.D));
}
// Distance from which a tile's bias is one number that is added behind the maximum of its scores: the table's range, or none where a number at
// its ends is -inf (which hides the tile) or too large to be held in fp32 together with a score: there the maximum has to be that of the rounded sums.
__device__ __forceinline__ int seq_bias_far(const SeqArgs& a, int h) {
    return __builtin_amdgcn_readfirstlane(fabsf(seq_bias_of(a, h, -a.D)) < SEQ_BIG && fabsf(seq_bias_of(a, h, a.D)) < SEQ_BIG ? a.D : 1 << 30);
}
// Statistics of rows in the backward pass. p = exp2(x - lse) needs lse = m + log2(l) to a fraction of one; where the row's maximum m is large (a table's
// lowest values, very large scores) fp32 drops log2(l) beside it, and p would be n times too large for n equal keys. For such rows the maximum and
// log2 of the sum are made anew, once, from the scores as the tile loops round them, and kept as two numbers: p = exp2((x - m) - log2 l).
__device__ __forceinline__ bool seq_row_big(float lse2) { return fabsf(lse2) >= SEQ_BIG && lse2 != INFINITY; }
// (x - m) - lg, with x - m held to what a maximum leaves; NaN stays
__device__ __forceinline__ float seq_exponent(float x, float m, float lg) { const float y = x - m; return (y > 0.f ? 0.f : y) - lg; }
// m and lg of the 16 rows that a wave holds in qf (row l15 at position p0 + l15), over the keys below kend; straight from memory: a rare path
template <typename T, int KS, bool BIAS>
__device__ __forceinline__ void seq_row_stats(const SeqArgs& a, const T* K, const unsigned char* mask, int kend, int h, int p0, const SeqFrag<T> (&qf)[KS], int l15, int g, float& m, float& lg) {
    float mx = -INFINITY, l = 0.f;
    for (int k0 = 0; k0 < kend; k0 += 16) {
        const int key = k0 + l15;
        const bool in = key < kend && (!mask || mask[key] != 0);
        f32x4 x = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int s = 0; s < KS; ++s) x = seq_mma(seq_frag_row<T>(K + (long)key * a.k.row, in, s, g, a.d), qf[s], x);
        const unsigned seen = (unsigned)__ballot(in) >> (4 * g);
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            const int rel = k0 + 4 * g + r - p0 - l15;
            const float b = BIAS ? seq_bias_of(a, h, min(max(rel, -a.D), a.D)) : 0.f;
            x[r] = ((seen >> r) & 1) && (!a.causal || rel <= 0) ? __builtin_fmaf(x[r], a.scale * SEQ_L2E, b) : -INFINITY;
        }
        const float mn = fmaxf(mx, seq_group_max(fmaxf(fmaxf(x[0], x[1]), fmaxf(x[2], x[3])))), off = mn == -INFINITY ? 0.f : mn;
        l *= __builtin_amdgcn_exp2f(mx - off);
#pragma unroll
        for (int r = 0; r < 4; ++r) l += __builtin_amdgcn_exp2f(x[r] - off);
        mx = mn;
    }
    m = mx == -INFINITY ? INFINITY : mx;          // (nothing visible: probabilities of zero)
    lg = mx == -INFINITY ? 0.f : __builtin_amdgcn_logf(seq_group_sum(l));
}
// Visible rows of a tile as a bit mask (wave-uniform): rows at or beyond `len` and rows that the key mask hides are clear. The mask's byte of this
// lane's row is fetched a tile ahead (seq_mask_byte), so that its latency is not paid between two tiles.
template <int TK> __device__ __forceinline__ int seq_mask_byte(const unsigned char* mask, int r0, int len, int lane) {
    const int r = r0 + lane;
    return mask && lane < TK && r < len ? mask[r] : 0;
}
template <int TK> __device__ __forceinline__ unsigned long long seq_live(bool masked, int byte, int r0, int len) {
    if (masked) return __ballot(byte != 0);
    const int n = len - r0;
    return n >= 64 ? SEQ_ALL<TK> : (n <= 0 ? 0ull : (((1ull << n) - 1) & SEQ_ALL<TK>));
}
__device__ __forceinline__ int seq_clamp_len(const int* p, int b, int n) { return p ? min(max(p[b], 0), n) : n; }
__device__ __forceinline__ int seq_pos(const int* p, int b) { return p ? min(max(p[b], -SEQ_POS_LIM), SEQ_POS_LIM) : 0; }
// block id -> (rank of the block along its axis, sample x head). Ranks are the slow index, so that with a causal mask the blocks with the most
// work start first whatever their head; samples and key / value heads are the fast one: blocks are dealt to the 8 XCDs in turn, so the blocks
// that read one key / value head meet in one L2 wherever B * Hkv is a multiple of 8, and the query heads that share it lie B * Hkv apart.
__device__ __forceinline__ void seq_item(const SeqArgs& a, int id, int& rank, int& b, int& h) {
    const int n = a.B * a.Hkv, all = n * a.G;
    rank = id / all;
    const int x = id - rank * all, gi = x / n, bk = x - gi * n;
    b = bk / a.Hkv;
    h = (bk - b * a.Hkv) * a.G + gi;
}
// The same for kernels bound by the rows of Q: the heads of a token lie side by side in memory, and a head of 40 or 80 elements ends inside a
// 128-byte line, so the blocks of all heads of one (sample, rank) go to one XCD, one after the other. Ids past the last item: false.
__device__ __forceinline__ bool seq_item_by_row(int B, int H, int ranks, int id, int& rank, int& b, int& h) {
    const int x = id & 7, y = id >> 3, u = y / H * 8 + x;
    h = y - y / H * H;
    rank = u / B; b = u - rank * B;
    return u < B * ranks;
}
inline unsigned seq_grid_by_row(long B, long H, long ranks) { return (unsigned)(cdiv(B * ranks, 8) * 8 * H); }
#endif  // __HIPCC__

#define SEQ_DT_SWITCH(d, DTC, ...)                                   \
    do {                                                             \
        if ((d) <= 32) { constexpr int DTC = 2; __VA_ARGS__; }       \
        else if ((d) <= 48) { constexpr int DTC = 3; __VA_ARGS__; }  \
        else if ((d) <= 64) { constexpr int DTC = 4; __VA_ARGS__; }  \
        else if ((d) <= 80) { constexpr int DTC = 5; __VA_ARGS__; }  \
        else if ((d) <= 128) { constexpr int DTC = 8; __VA_ARGS__; } \
        else { constexpr int DTC = 10; __VA_ARGS__; }                \
    } while (0)

}  // namespace cb
