// Attention for training: forward with the log-sum-exp of every row, and a backward pass that recomputes the probabilities from it.
//   s_ij = scale q_i . k_j,  lse_i = log sum_j exp s_ij,  p_ij = exp(s_ij - lse_i),  o_i = sum_j p_ij v_j
//   D_i = do_i . o_i,  ds_ij = p_ij (do_i . v_j - D_i),  dq_i = scale sum_j ds_ij k_j,  dk_j = scale sum_i ds_ij q_i,  dv_j = sum_i p_ij do_i
// over the keys j that query i may attend to.  Nothing of size Lq x Lk is stored.
//
// All three passes are one structure: a wave owns 16 NQ columns (queries in the forward and dq passes, keys in the dk / dv pass) whose
// operands stay in registers, and walks the other axis in tiles that the workgroup stages through LDS.  The scores are computed
// transposed (rows = the walked axis), so that the accumulator of the first product, lane column i and rows 4 g + 0..3, is already
// the B operand of the second: two 16-row tiles give a lane 8 contraction slots, and the matching A operand (the walked tensor with its
// rows as contraction) comes from the same LDS tile through the transposing read.  The probabilities never leave registers.
// The dq and the dk / dv pass each recompute the scores (14 instead of 10 D flops per pair): no atomics, the same bits every run.
#include "tb_ops.hpp"

#include "tb_ops_host.hpp"

namespace tb {
namespace op {

namespace {

constexpr float NEG_INF = -__builtin_inff();

// workgroup -> (row of the (batch, head) list, tile of the columns x split).  Workgroups go to the eight XCDs round robin; with
// `xcd` all tiles of one (batch, head) land on the same XCD, whose L2 then holds its keys and values once.
__device__ __forceinline__ bool decode(unsigned id, int n_inner, int n_bh, int xcd, int& bh, int& inner) {
    if (xcd) {
        const unsigned lo = id & 7u, r = id >> 3;
        inner = (int)(r % (unsigned)n_inner);
        bh = (int)(r / (unsigned)n_inner) * 8 + (int)lo;
    } else {
        inner = (int)(id % (unsigned)n_inner);
        bh = (int)(id / (unsigned)n_inner);
    }
    return bh < n_bh;
}

// A tile of KT rows x D columns on its way from global memory to LDS: every thread holds PT chunks of 8 elements.
template <typename T, int DP, int NT, int KT>
struct Stage {
    static constexpr int NP = Planes<T>::N, CH = DP / 8, PT = (KT * CH + NT - 1) / NT, LD = DP + LDS_PAD;
    Held<T> r[PT];
    // rows row0 .. row0 + KT - 1 of `base` (row stride `ld`); a row outside [0, end) or marked invalid becomes zero, whatever it holds
    __device__ __forceinline__ void load(const T* base, int64_t ld, const uint8_t* valid, int row0, int end, int D, int tid) {
#pragma unroll
        for (int c = 0; c < PT; ++c) {
            const int idx = tid + c * NT, row = row0 + idx / CH, col = (idx % CH) * 8;
            r[c].zero();
            if (idx < KT * CH && row < end && col < D) {
                r[c].load(base + (int64_t)row * ld + col, D - col);
                if (valid && !valid[row]) r[c].zero();
            }
        }
    }
    __device__ __forceinline__ void store(bf16* lds, int tid) const {
#pragma unroll
        for (int c = 0; c < PT; ++c) {
            const int idx = tid + c * NT;
            if (KT * CH % NT == 0 || idx < KT * CH) {
                bf16x8 pl[NP];
                r[c].planes(pl);
#pragma unroll
                for (int n = 0; n < NP; ++n) *reinterpret_cast<bf16x8*>(lds + (size_t)n * KT * LD + (idx / CH) * LD + (idx % CH) * 8) = pl[n];
            }
        }
    }
};

// B operand of 16 columns: column i = row `row` of a [., D] matrix in global memory (zero where not `on`)
template <typename T, int KC>
__device__ __forceinline__ void load_columns(const T* row, bool on, int D, int lane, Frag<Planes<T>::N> (&f)[KC]) {
#pragma unroll
    for (int kc = 0; kc < KC; ++kc) {
        Held<T> h;
        h.zero();
        const int col = kc * 32 + 8 * (lane >> 4);
        if (on && col < D) h.load(row + col, D - col);
        h.planes(f[kc].p);
    }
}

// two 16-row accumulator tiles -> the B operand of the second product (k slots 8 g + 0..3 from the first tile, 4..7 from the second)
template <int NP>
__device__ __forceinline__ void as_operand(const f32x4& a, const f32x4& b, Frag<NP>& f) {
    const float x[8] = {a[0], a[1], a[2], a[3], b[0], b[1], b[2], b[3]};
    to_planes<NP>(x, f.p);
}

// ------------------------------------------------------------------------------------------------ forward
template <typename T, int DP, int NW, int NQ, int KT>
__global__ __launch_bounds__(64 * NW) void k_attn_fwd(const AttnP p) {
    constexpr int NP = Planes<T>::N, KC = DP / 32, DN = DP / 16, KN = KT / 16, NT = 64 * NW, LD = DP + LDS_PAD, QT = 16 * NQ * NW;
    __shared__ __attribute__((aligned(16))) bf16 lk[NP * KT * LD];
    __shared__ __attribute__((aligned(16))) bf16 lv[NP * KT * LD];
    __shared__ __attribute__((aligned(16))) float lb[KT];
    int bh, inner;
    if (!decode(blockIdx.x, p.n_col_tile * p.n_split, p.B * p.H, p.xcd, bh, inner)) return;
    const int split = inner / p.n_col_tile, qt = p.n_col_tile - 1 - inner % p.n_col_tile;  // (causal: the longest walks first)
    const int b = bh / p.H, h = bh % p.H, hk = h / p.G;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, i16 = lane & 15, g = lane >> 4;
    const int qb = qt * QT, q0 = qb + wave * 16 * NQ, off = p.Lk - p.Lq;
    const T* kp = (const T*)p.k + b * p.ks[0] + hk * p.ks[2];
    const T* vp = (const T*)p.v + b * p.vs[0] + hk * p.vs[2];
    const uint8_t* kvalid = p.key_valid ? p.key_valid + (int64_t)b * p.Lk : nullptr;

    Frag<NP> qf[NQ][KC];
    int qi[NQ];
#pragma unroll
    for (int n = 0; n < NQ; ++n) {
        qi[n] = q0 + n * 16 + i16;
        const bool on = qi[n] < p.Lq && (!p.query_valid || p.query_valid[(int64_t)b * p.Lq + qi[n]]);
        load_columns<T, KC>((const T*)p.q + b * p.qs[0] + (int64_t)(on ? qi[n] : 0) * p.qs[1] + h * p.qs[2], on, p.D, lane, qf[n]);
    }
    f32x4 acc[NQ][DN];
    float m[NQ], l[NQ];
#pragma unroll
    for (int n = 0; n < NQ; ++n) {
        m[n] = NEG_INF;
        l[n] = 0.f;
#pragma unroll
        for (int d = 0; d < DN; ++d) acc[n][d] = (f32x4){0.f, 0.f, 0.f, 0.f};
    }
    int j0 = split * p.split_len, jend = min(p.Lk, j0 + p.split_len);
    if (p.causal) jend = min(jend, min(p.Lq, qb + QT) + off);

    Stage<T, DP, NT, KT> sk, sv;
    if (j0 < jend) {
        sk.load(kp, p.ks[1], kvalid, j0, jend, p.D, tid);
        sv.load(vp, p.vs[1], kvalid, j0, jend, p.D, tid);
    }
    for (; j0 < jend; j0 += KT) {
        __syncthreads();
        sk.store(lk, tid);
        sv.store(lv, tid);
        if (tid < KT) lb[tid] = (j0 + tid < jend && (!kvalid || kvalid[j0 + tid])) ? 0.f : NEG_INF;
        __syncthreads();
        if (j0 + KT < jend) {
            sk.load(kp, p.ks[1], kvalid, j0 + KT, jend, p.D, tid);
            sv.load(vp, p.vs[1], kvalid, j0 + KT, jend, p.D, tid);
        }
        f32x4 s[NQ][KN];
#pragma unroll
        for (int t = 0; t < KN; ++t) {
#pragma unroll
            for (int n = 0; n < NQ; ++n) s[n][t] = (f32x4){0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int kc = 0; kc < KC; ++kc) {
                Frag<NP> a;
                frag_rows<NP, LD>(lk, (size_t)KT * LD, t * 16, kc * 32, lane, a);
#pragma unroll
                for (int n = 0; n < NQ; ++n) s[n][t] = mma<NP>(a, qf[n][kc], s[n][t]);
            }
        }
        const bool biased = kvalid || j0 + KT > jend, diagonal = p.causal && j0 + KT - 1 > q0 + off;
#pragma unroll
        for (int n = 0; n < NQ; ++n) {
            float mx = NEG_INF;
#pragma unroll
            for (int t = 0; t < KN; ++t) {
                s[n][t] *= p.scale2;
                if (biased) s[n][t] += *reinterpret_cast<const f32x4*>(lb + t * 16 + 4 * g);
                if (diagonal) {
#pragma unroll
                    for (int e = 0; e < 4; ++e)
                        if (j0 + t * 16 + 4 * g + e > qi[n] + off) s[n][t][e] = NEG_INF;
                }
                if (p.mask && qi[n] < p.Lq) {
                    const uint8_t* mr = p.mask + b * p.mask_s[0] + (int64_t)qi[n] * p.mask_s[1] + j0 + t * 16 + 4 * g;
#pragma unroll
                    for (int e = 0; e < 4; ++e)
                        if (j0 + t * 16 + 4 * g + e < jend && mr[e]) s[n][t][e] = NEG_INF;
                }
#pragma unroll
                for (int e = 0; e < 4; ++e) mx = fmaxf(mx, s[n][t][e]);
            }
            mx = fmaxf(m[n], max_over_groups(mx));
            const float ref = mx == NEG_INF ? 0.f : mx;  // nothing to see yet: exp2(-inf - 0) = 0
            const float alpha = __builtin_amdgcn_exp2f(m[n] - ref);
            m[n] = mx;
            l[n] *= alpha;
#pragma unroll
            for (int d = 0; d < DN; ++d) acc[n][d] *= alpha;
#pragma unroll
            for (int t = 0; t < KN; ++t)
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    s[n][t][e] = __builtin_amdgcn_exp2f(s[n][t][e] - ref);
                    l[n] += s[n][t][e];
                }
        }
#pragma unroll
        for (int t = 0; t < KN; t += 2) {
            Frag<NP> pf[NQ];
#pragma unroll
            for (int n = 0; n < NQ; ++n) as_operand<NP>(s[n][t], s[n][t + 1], pf[n]);
#pragma unroll
            for (int d = 0; d < DN; ++d) {
                Frag<NP> a;
                frag_cols<NP, LD>(lv, (size_t)KT * LD, t * 16 + 4 * g, (t + 1) * 16 + 4 * g, d * 16, lane, a);
#pragma unroll
                for (int n = 0; n < NQ; ++n) acc[n][d] = mma<NP>(a, pf[n], acc[n][d]);
            }
        }
    }
#pragma unroll
    for (int n = 0; n < NQ; ++n) {
        const float sum = sum_over_groups(l[n]);
        if (qi[n] >= p.Lq) continue;
        const bool on = sum > 0.f || sum != sum;  // (a NaN row stays NaN)
        const bool valid = !p.query_valid || p.query_valid[(int64_t)b * p.Lq + qi[n]];
        const float inv = on && valid ? 1.f / sum : 0.f;
        const float lse2 = on && valid ? m[n] + __builtin_amdgcn_logf(sum) : NEG_INF;
        const int64_t row = (int64_t)bh * p.Lq + qi[n];
#pragma unroll
        for (int d = 0; d < DN; ++d) {
            const int col = d * 16 + 4 * g;
            f32x4 o = acc[n][d] * inv;
            if (!(on && valid)) o = (f32x4){0.f, 0.f, 0.f, 0.f};
            if (col >= p.D) continue;
            if (p.n_split > 1)
                store4(p.part + ((int64_t)split * p.B * p.H * p.Lq + row) * p.D + col, p.D - col, o);
            else
                store4((T*)p.out + b * p.os[0] + qi[n] * p.os[1] + h * p.os[2] + col, p.D - col, o);
        }
        if (g == 0) {
            if (p.n_split > 1)
                p.part_lse[(int64_t)split * p.B * p.H * p.Lq + row] = lse2;
            else
                p.lse[row] = lse2 * LN2;
        }
    }
}

// join of the splits: o = sum_s 2^(lse_s - lse) o_s.  One thread per 4 columns of a row.
template <typename T>
__global__ __launch_bounds__(256) void k_attn_join(const AttnP p) {
    const int cols = (p.D + 3) / 4;
    const int64_t id = (int64_t)blockIdx.x * 256 + threadIdx.x, rows = (int64_t)p.B * p.H * p.Lq, row = id / cols;
    if (row >= rows) return;
    const int col = (int)(id % cols) * 4, q = (int)(row % p.Lq), h = (int)(row / p.Lq % p.H);
    const int64_t b = row / p.Lq / p.H;
    float m = NEG_INF;
    for (int s = 0; s < p.n_split; ++s) m = fmaxf(m, p.part_lse[s * rows + row]);
    const float ref = m == NEG_INF ? 0.f : m;
    float sum = 0.f;
    f32x4 o = {0.f, 0.f, 0.f, 0.f};
    for (int s = 0; s < p.n_split; ++s) {
        const float w = __builtin_amdgcn_exp2f(p.part_lse[s * rows + row] - ref);
        const float* src = p.part + (s * rows + row) * p.D + col;
        sum += w;
#pragma unroll
        for (int e = 0; e < 4; ++e)
            if (col + e < p.D) o[e] = __builtin_fmaf(w, src[e], o[e]);
    }
    const bool on = sum > 0.f || sum != sum;
    o = on ? o * (1.f / sum) : (f32x4){0.f, 0.f, 0.f, 0.f};
    store4((T*)p.out + b * p.os[0] + q * p.os[1] + h * p.os[2] + col, p.D - col, o);
    if (col == 0) p.lse[row] = on ? (ref + __builtin_amdgcn_logf(sum)) * LN2 : NEG_INF;
}

// ------------------------------------------------------------------------------------------------ backward: dq
template <typename T, int DP, int NW, int NQ, int KT>
__global__ __launch_bounds__(64 * NW) void k_attn_dq(const AttnP p) {
    constexpr int NP = Planes<T>::N, KC = DP / 32, DN = DP / 16, KN = KT / 16, NT = 64 * NW, LD = DP + LDS_PAD, QT = 16 * NQ * NW;
    __shared__ __attribute__((aligned(16))) bf16 lk[NP * KT * LD];
    __shared__ __attribute__((aligned(16))) bf16 lv[NP * KT * LD];
    __shared__ __attribute__((aligned(16))) float lb[KT];
    int bh, inner;
    if (!decode(blockIdx.x, p.n_col_tile * p.n_split, p.B * p.H, p.xcd, bh, inner)) return;
    const int split = inner / p.n_col_tile, qt = p.n_col_tile - 1 - inner % p.n_col_tile;
    const int b = bh / p.H, h = bh % p.H, hk = h / p.G;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, i16 = lane & 15, g = lane >> 4;
    const int qb = qt * QT, q0 = qb + wave * 16 * NQ, off = p.Lk - p.Lq;
    const T* kp = (const T*)p.k + b * p.ks[0] + hk * p.ks[2];
    const T* vp = (const T*)p.v + b * p.vs[0] + hk * p.vs[2];
    const uint8_t* kvalid = p.key_valid ? p.key_valid + (int64_t)b * p.Lk : nullptr;

    Frag<NP> qf[NQ][KC], gf[NQ][KC];
    int qi[NQ];
    float nlse[NQ], delta[NQ];
    f32x4 acc[NQ][DN];
#pragma unroll
    for (int n = 0; n < NQ; ++n) {
        qi[n] = q0 + n * 16 + i16;
        const bool in = qi[n] < p.Lq, on = in && (!p.query_valid || p.query_valid[(int64_t)b * p.Lq + qi[n]]);
        const int64_t qr = on ? qi[n] : 0, row = (int64_t)bh * p.Lq + qi[n];
        const T* dop = (const T*)p.d_out + b * p.dos[0] + qr * p.dos[1] + h * p.dos[2];
        load_columns<T, KC>((const T*)p.q + b * p.qs[0] + qr * p.qs[1] + h * p.qs[2], on, p.D, lane, qf[n]);
        load_columns<T, KC>(dop, on, p.D, lane, gf[n]);
        const T* op = (const T*)p.out + b * p.os[0] + qr * p.os[1] + h * p.os[2];
        float dot = 0.f;
#pragma unroll
        for (int kc = 0; kc < KC; ++kc) {
            const int col = kc * 32 + 8 * g;
            if (on && col < p.D) {
                float x[8], y[8];
                load8(dop + col, p.D - col, x);
                load8(op + col, p.D - col, y);
#pragma unroll
                for (int e = 0; e < 8; ++e) dot = __builtin_fmaf(x[e], y[e], dot);
            }
        }
        delta[n] = sum_over_groups(dot);
        const float lse = on ? p.lse[row] : NEG_INF;
        nlse[n] = lse == NEG_INF ? NEG_INF : -lse * LOG2E;  // an empty row: p = 2^(-inf) = 0
        if (in && g == 0 && split == 0) p.delta[row] = delta[n];
#pragma unroll
        for (int d = 0; d < DN; ++d) acc[n][d] = (f32x4){0.f, 0.f, 0.f, 0.f};
    }
    int j0 = split * p.split_len, jend = min(p.Lk, j0 + p.split_len);
    if (p.causal) jend = min(jend, min(p.Lq, qb + QT) + off);
    Stage<T, DP, NT, KT> sk, sv;
    if (j0 < jend) {
        sk.load(kp, p.ks[1], kvalid, j0, jend, p.D, tid);
        sv.load(vp, p.vs[1], kvalid, j0, jend, p.D, tid);
    }
    for (; j0 < jend; j0 += KT) {
        __syncthreads();
        sk.store(lk, tid);
        sv.store(lv, tid);
        if (tid < KT) lb[tid] = (j0 + tid < jend && (!kvalid || kvalid[j0 + tid])) ? 0.f : NEG_INF;
        __syncthreads();
        if (j0 + KT < jend) {
            sk.load(kp, p.ks[1], kvalid, j0 + KT, jend, p.D, tid);
            sv.load(vp, p.vs[1], kvalid, j0 + KT, jend, p.D, tid);
        }
        const bool biased = kvalid || j0 + KT > jend, diagonal = p.causal && j0 + KT - 1 > q0 + off;
#pragma unroll
        for (int t2 = 0; t2 < KN; t2 += 2) {
            f32x4 ds[NQ][2];
#pragma unroll
            for (int u = 0; u < 2; ++u) {
                const int t = t2 + u;
                f32x4 s[NQ], dp[NQ];
#pragma unroll
                for (int n = 0; n < NQ; ++n) s[n] = dp[n] = (f32x4){0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int kc = 0; kc < KC; ++kc) {
                    Frag<NP> a, v;
                    frag_rows<NP, LD>(lk, (size_t)KT * LD, t * 16, kc * 32, lane, a);
                    frag_rows<NP, LD>(lv, (size_t)KT * LD, t * 16, kc * 32, lane, v);
#pragma unroll
                    for (int n = 0; n < NQ; ++n) {
                        s[n] = mma<NP>(a, qf[n][kc], s[n]);
                        dp[n] = mma<NP>(v, gf[n][kc], dp[n]);
                    }
                }
#pragma unroll
                for (int n = 0; n < NQ; ++n) {
                    f32x4 x;
#pragma unroll
                    for (int e = 0; e < 4; ++e) x[e] = __builtin_fmaf(s[n][e], p.scale2, nlse[n]);
                    if (biased) x += *reinterpret_cast<const f32x4*>(lb + t * 16 + 4 * g);
                    if (diagonal) {
#pragma unroll
                        for (int e = 0; e < 4; ++e)
                            if (j0 + t * 16 + 4 * g + e > qi[n] + off) x[e] = NEG_INF;
                    }
                    if (p.mask && qi[n] < p.Lq) {
                        const uint8_t* mr = p.mask + b * p.mask_s[0] + (int64_t)qi[n] * p.mask_s[1] + j0 + t * 16 + 4 * g;
#pragma unroll
                        for (int e = 0; e < 4; ++e)
                            if (j0 + t * 16 + 4 * g + e < jend && mr[e]) x[e] = NEG_INF;
                    }
#pragma unroll
                    for (int e = 0; e < 4; ++e) ds[n][u][e] = __builtin_amdgcn_exp2f(x[e]) * (dp[n][e] - delta[n]);
                }
            }
            Frag<NP> df[NQ];
#pragma unroll
            for (int n = 0; n < NQ; ++n) as_operand<NP>(ds[n][0], ds[n][1], df[n]);
#pragma unroll
            for (int d = 0; d < DN; ++d) {
                Frag<NP> a;
                frag_cols<NP, LD>(lk, (size_t)KT * LD, t2 * 16 + 4 * g, (t2 + 1) * 16 + 4 * g, d * 16, lane, a);
#pragma unroll
                for (int n = 0; n < NQ; ++n) acc[n][d] = mma<NP>(a, df[n], acc[n][d]);
            }
        }
    }
#pragma unroll
    for (int n = 0; n < NQ; ++n) {
        if (qi[n] >= p.Lq) continue;
#pragma unroll
        for (int d = 0; d < DN; ++d) {
            const int col = d * 16 + 4 * g;
            if (col >= p.D) continue;
            const f32x4 o = acc[n][d] * p.scale;
            if (p.n_split > 1)
                store4(p.part + (((int64_t)split * p.B * p.Lq + (int64_t)b * p.Lq + qi[n]) * p.H + h) * p.D + col, p.D - col, o);
            else
                store4((T*)p.dq + b * p.dqs[0] + qi[n] * p.dqs[1] + h * p.dqs[2] + col, p.D - col, o);
        }
    }
}

// ------------------------------------------------------------------------------------------------ backward: dk, dv
// Columns are keys; the walk goes over the query tiles of every head of the key's group, so the gradients of shared heads are summed
// in registers.  A split takes a contiguous part of that walk.
template <typename T, int DP, int NW, int NQ, int KT>
__global__ __launch_bounds__(64 * NW) void k_attn_dkv(const AttnP p) {
    constexpr int NP = Planes<T>::N, KC = DP / 32, DN = DP / 16, KN = KT / 16, NT = 64 * NW, LD = DP + LDS_PAD, CT = 16 * NQ * NW;
    __shared__ __attribute__((aligned(16))) bf16 lq[NP * KT * LD];
    __shared__ __attribute__((aligned(16))) bf16 lg[NP * KT * LD];
    __shared__ __attribute__((aligned(16))) float ll[KT];
    __shared__ __attribute__((aligned(16))) float ld[KT];
    int bh, inner;
    if (!decode(blockIdx.x, p.n_col_tile * p.n_split, p.B * p.Hkv, p.xcd, bh, inner)) return;
    const int split = inner / p.n_col_tile, kt = inner % p.n_col_tile;  // (causal: the first keys have the longest walks)
    const int b = bh / p.Hkv, hk = bh % p.Hkv;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, i16 = lane & 15, g = lane >> 4;
    const int kb = kt * CT, k0 = kb + wave * 16 * NQ, off = p.Lk - p.Lq;
    const uint8_t* qvalid = p.query_valid ? p.query_valid + (int64_t)b * p.Lq : nullptr;

    Frag<NP> kf[NQ][KC], vf[NQ][KC];
    int ki[NQ];
    bool on[NQ];
    f32x4 dk[NQ][DN], dv[NQ][DN];
#pragma unroll
    for (int n = 0; n < NQ; ++n) {
        ki[n] = k0 + n * 16 + i16;
        on[n] = ki[n] < p.Lk && (!p.key_valid || p.key_valid[(int64_t)b * p.Lk + ki[n]]);
        const int64_t kr = on[n] ? ki[n] : 0;
        load_columns<T, KC>((const T*)p.k + b * p.ks[0] + kr * p.ks[1] + hk * p.ks[2], on[n], p.D, lane, kf[n]);
        load_columns<T, KC>((const T*)p.v + b * p.vs[0] + kr * p.vs[1] + hk * p.vs[2], on[n], p.D, lane, vf[n]);
#pragma unroll
        for (int d = 0; d < DN; ++d) dk[n][d] = dv[n][d] = (f32x4){0.f, 0.f, 0.f, 0.f};
    }
    // the walk: step t = (head of the group, query tile), query tiles from the first one that sees a key of this tile
    const int n_qt = (p.Lq + KT - 1) / KT, first = p.causal ? min(n_qt, max(0, kb - off) / KT) : 0, per_head = n_qt - first;
    const int n_step = p.G * per_head, len = (n_step + p.n_split - 1) / p.n_split;
    int t = split * len;
    const int tend = min(n_step, t + len);

    Stage<T, DP, NT, KT> sq, sg;
    float r_lse = 0.f, r_delta = 0.f;
    auto load = [&](int step) {
        const int h = hk * p.G + step / per_head, q0 = (first + step % per_head) * KT;
        sq.load((const T*)p.q + b * p.qs[0] + h * p.qs[2], p.qs[1], qvalid, q0, p.Lq, p.D, tid);
        sg.load((const T*)p.d_out + b * p.dos[0] + h * p.dos[2], p.dos[1], qvalid, q0, p.Lq, p.D, tid);
        if (tid < KT) {
            const bool in = q0 + tid < p.Lq && (!qvalid || qvalid[q0 + tid]);
            const int64_t row = ((int64_t)b * p.H + h) * p.Lq + q0 + tid;
            const float lse = in ? p.lse[row] : NEG_INF;
            r_lse = lse == NEG_INF ? NEG_INF : -lse * LOG2E;
            r_delta = in ? p.delta[row] : 0.f;
        }
    };
    if (t < tend) load(t);
    for (; t < tend; ++t) {
        __syncthreads();
        sq.store(lq, tid);
        sg.store(lg, tid);
        if (tid < KT) {
            ll[tid] = r_lse;
            ld[tid] = r_delta;
        }
        __syncthreads();
        const int q0 = (first + t % per_head) * KT;
        if (t + 1 < tend) load(t + 1);
        const bool diagonal = p.causal && k0 + 16 * NQ - 1 > q0 + off;
#pragma unroll
        for (int t2 = 0; t2 < KN; t2 += 2) {
            f32x4 pr[NQ][2], ds[NQ][2];
#pragma unroll
            for (int u = 0; u < 2; ++u) {
                const int tt = t2 + u;
                f32x4 s[NQ], dp[NQ];
#pragma unroll
                for (int n = 0; n < NQ; ++n) s[n] = dp[n] = (f32x4){0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int kc = 0; kc < KC; ++kc) {
                    Frag<NP> a, v;
                    frag_rows<NP, LD>(lq, (size_t)KT * LD, tt * 16, kc * 32, lane, a);
                    frag_rows<NP, LD>(lg, (size_t)KT * LD, tt * 16, kc * 32, lane, v);
#pragma unroll
                    for (int n = 0; n < NQ; ++n) {
                        s[n] = mma<NP>(a, kf[n][kc], s[n]);
                        dp[n] = mma<NP>(v, vf[n][kc], dp[n]);
                    }
                }
                const f32x4 nl = *reinterpret_cast<const f32x4*>(ll + tt * 16 + 4 * g), de = *reinterpret_cast<const f32x4*>(ld + tt * 16 + 4 * g);
#pragma unroll
                for (int n = 0; n < NQ; ++n) {
                    f32x4 x;
#pragma unroll
                    for (int e = 0; e < 4; ++e) x[e] = __builtin_fmaf(s[n][e], p.scale2, nl[e]);
                    if (diagonal) {
#pragma unroll
                        for (int e = 0; e < 4; ++e)
                            if (ki[n] > q0 + tt * 16 + 4 * g + e + off) x[e] = NEG_INF;
                    }
                    if (p.mask && ki[n] < p.Lk) {
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            const int q = q0 + tt * 16 + 4 * g + e;
                            if (q < p.Lq && p.mask[b * p.mask_s[0] + (int64_t)q * p.mask_s[1] + ki[n]]) x[e] = NEG_INF;
                        }
                    }
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        pr[n][u][e] = __builtin_amdgcn_exp2f(x[e]);
                        ds[n][u][e] = pr[n][u][e] * (dp[n][e] - de[e]);
                    }
                }
            }
            Frag<NP> pf[NQ], df[NQ];
#pragma unroll
            for (int n = 0; n < NQ; ++n) {
                as_operand<NP>(pr[n][0], pr[n][1], pf[n]);
                as_operand<NP>(ds[n][0], ds[n][1], df[n]);
            }
#pragma unroll
            for (int d = 0; d < DN; ++d) {
                Frag<NP> a, v;
                frag_cols<NP, LD>(lg, (size_t)KT * LD, t2 * 16 + 4 * g, (t2 + 1) * 16 + 4 * g, d * 16, lane, a);
                frag_cols<NP, LD>(lq, (size_t)KT * LD, t2 * 16 + 4 * g, (t2 + 1) * 16 + 4 * g, d * 16, lane, v);
#pragma unroll
                for (int n = 0; n < NQ; ++n) {
                    dv[n][d] = mma<NP>(a, pf[n], dv[n][d]);
                    dk[n][d] = mma<NP>(v, df[n], dk[n][d]);
                }
            }
        }
    }
#pragma unroll
    for (int n = 0; n < NQ; ++n) {
        if (ki[n] >= p.Lk) continue;
#pragma unroll
        for (int d = 0; d < DN; ++d) {
            const int col = d * 16 + 4 * g;
            if (col >= p.D) continue;
            const f32x4 zero = {0.f, 0.f, 0.f, 0.f}, ok = on[n] ? dk[n][d] * p.scale : zero, ov = on[n] ? dv[n][d] : zero;
            if (p.n_split > 1) {
                const int64_t at = (((int64_t)split * p.B * p.Lk + (int64_t)b * p.Lk + ki[n]) * p.Hkv + hk) * p.D + col;
                store4(p.part + at, p.D - col, ok);
                store4(p.part + (int64_t)p.n_split * p.B * p.Lk * p.Hkv * p.D + at, p.D - col, ov);
            } else {
                store4((T*)p.dk + b * p.dks[0] + ki[n] * p.dks[1] + hk * p.dks[2] + col, p.D - col, ok);
                store4((T*)p.dv + b * p.dvs[0] + ki[n] * p.dvs[1] + hk * p.dvs[2] + col, p.D - col, ov);
            }
        }
    }
}

// sum of the splits' gradients, in split order, into a strided [B, L, H, D] tensor
template <typename T>
__global__ __launch_bounds__(256) void k_attn_sum(const float* part, int n_split, int B, int L, int H, int D, T* dst, int64_t sb, int64_t sl, int64_t sh) {
    const int cols = (D + 3) / 4;
    const int64_t id = (int64_t)blockIdx.x * 256 + threadIdx.x, rows = (int64_t)B * L * H, row = id / cols;
    if (row >= rows) return;
    const int col = (int)(id % cols) * 4;
    f32x4 o = {0.f, 0.f, 0.f, 0.f};
    for (int s = 0; s < n_split; ++s) {
        const float* src = part + (s * rows + row) * D + col;
#pragma unroll
        for (int e = 0; e < 4; ++e)
            if (col + e < D) o[e] += src[e];
    }
    const int64_t h = row % H, l = row / H % L, b = row / H / L;
    store4(dst + b * sb + l * sl + h * sh + col, D - col, o);
}

enum Pass { FWD, DQ, DKV };

struct Shape {  // of one launch: columns per workgroup, walked rows per tile
    int col_tile, walk_tile;
    void (*kernel)(AttnP);
    int threads;
};

template <typename T, int DP, int NW, int NQ, int KT>
Shape shape(Pass pass) {
    return {16 * NQ * NW, KT, pass == FWD ? k_attn_fwd<T, DP, NW, NQ, KT> : pass == DQ ? k_attn_dq<T, DP, NW, NQ, KT> : k_attn_dkv<T, DP, NW, NQ, KT>, 64 * NW};
}

template <typename T, int DP>
Shape choose(Pass pass, int n_col) {
    constexpr int KT = sizeof(T) == 2 ? 64 : DP <= 64 ? 32 : 32;
    if (n_col <= 16) return shape<T, DP, 1, 1, 32>(pass);
    if (n_col <= 32) return shape<T, DP, 1, 2, 32>(pass);
    return shape<T, DP, 4, 1, KT>(pass);
}

Shape choose(const AttnP& p, Pass pass) {
    const int n_col = pass == DKV ? p.Lk : p.Lq;
    if (p.dtype == 1) return p.D <= 32 ? choose<bf16, 32>(pass, n_col) : p.D <= 64 ? choose<bf16, 64>(pass, n_col) : choose<bf16, 128>(pass, n_col);
    return p.D <= 32 ? choose<float, 32>(pass, n_col) : p.D <= 64 ? choose<float, 64>(pass, n_col) : choose<float, 128>(pass, n_col);
}

// Few workgroups and a long walk: the walk is split over workgroups whose results a second kernel joins, until the chip has about two
// workgroups per CU; a part keeps at least four tiles.
struct Plan {
    Shape s;
    int n_col_tile, n_split, split_len;
    int64_t n_bh, blocks;
};
Plan plan(const AttnP& p, Pass pass) {
    Plan r;
    r.s = choose(p, pass);
    const int n_col = pass == DKV ? p.Lk : p.Lq;
    r.n_col_tile = (n_col + r.s.col_tile - 1) / r.s.col_tile;
    r.n_bh = (int64_t)p.B * (pass == DKV ? p.Hkv : p.H);
    const int walk = pass == DKV ? p.Lq : p.Lk;
    const int64_t tiles = (int64_t)((walk + r.s.walk_tile - 1) / r.s.walk_tile) * (pass == DKV ? p.G : 1);
    const int64_t base = r.n_bh * r.n_col_tile, waves = 512 * 4 / (r.s.threads / 64);
    int64_t n = base * 2 <= waves ? waves / (base > 0 ? base : 1) : 1;
    n = n < tiles / 4 ? n : tiles / 4;
    if (n < 1) n = 1;
    if (n > 64) n = 64;
    r.split_len = (int)((tiles + n - 1) / n) * r.s.walk_tile;  // (DKV: the kernel cuts its own walk, only n_split counts)
    r.n_split = pass == DKV ? (int)n : (int)((walk + r.split_len - 1) / (r.split_len > 0 ? r.split_len : 1));
    if (r.n_split < 1) r.n_split = 1;
    if (r.split_len < 1) r.split_len = r.s.walk_tile;
    r.blocks = base * r.n_split;
    return r;
}

int64_t part_floats(const AttnP& p, Pass pass, int n_split) {
    if (n_split <= 1) return 0;
    if (pass == FWD) return (int64_t)n_split * p.B * p.H * p.Lq * (p.D + 1);
    return pass == DQ ? (int64_t)n_split * p.B * p.Lq * p.H * p.D : 2 * (int64_t)n_split * p.B * p.Lk * p.Hkv * p.D;
}

const char* launch(AttnP p, Pass pass, const Plan& r, hipStream_t s) {
    p.n_col_tile = r.n_col_tile;
    p.n_split = r.n_split;
    p.split_len = r.split_len;
    p.xcd = r.n_bh % 8 == 0 && (int64_t)r.n_col_tile * r.n_split > 1;
    if (r.blocks <= 0) return nullptr;
    if (r.blocks > 0x7fffffff) return "too many workgroups (batch x heads x tiles > 2^31)";
    r.s.kernel<<<dim3((unsigned)r.blocks), dim3(r.s.threads), 0, s>>>(p);
    return nullptr;
}

template <typename T>
void launch_sum(const float* part, int n_split, int B, int L, int H, int D, void* dst, const int64_t* st, hipStream_t s) {
    const int64_t n = (int64_t)B * L * H * ((D + 3) / 4);
    k_attn_sum<T><<<dim3((unsigned)((n + 255) / 256)), dim3(256), 0, s>>>(part, n_split, B, L, H, D, (T*)dst, st[0], st[1], st[2]);
}

}  // namespace

int64_t attention_workspace(const AttnP& p, bool backward) {
    if (!backward) return 4 * part_floats(p, FWD, plan(p, FWD).n_split);
    const int64_t a = part_floats(p, DQ, plan(p, DQ).n_split), b = part_floats(p, DKV, plan(p, DKV).n_split);
    return 4 * ((int64_t)p.B * p.H * p.Lq + (a > b ? a : b));  // delta, and the parts of one pass after the other
}

const char* run_attention(AttnP p, float* ws, hipStream_t s) {
    const Plan r = plan(p, FWD);
    const int64_t rows = (int64_t)p.B * p.H * p.Lq;
    if (rows == 0) return nullptr;
    p.part = ws;
    p.part_lse = ws + (int64_t)r.n_split * rows * p.D;
    if (const char* e = launch(p, FWD, r, s)) return e;
    if (r.n_split > 1) {
        p.n_split = r.n_split;
        const unsigned blocks = (unsigned)((rows * ((p.D + 3) / 4) + 255) / 256);
        if (p.dtype == 1)
            k_attn_join<bf16><<<dim3(blocks), dim3(256), 0, s>>>(p);
        else
            k_attn_join<float><<<dim3(blocks), dim3(256), 0, s>>>(p);
    }
    return nullptr;
}

const char* run_attention_backward(AttnP p, float* ws, hipStream_t s) {
    p.delta = ws;
    p.part = ws + (int64_t)p.B * p.H * p.Lq;
    const Plan a = plan(p, DQ), b = plan(p, DKV);
    if (const char* e = launch(p, DQ, a, s)) return e;
    if (a.n_split > 1 && p.Lq > 0) {
        if (p.dtype == 1)
            launch_sum<bf16>(p.part, a.n_split, p.B, p.Lq, p.H, p.D, p.dq, p.dqs, s);
        else
            launch_sum<float>(p.part, a.n_split, p.B, p.Lq, p.H, p.D, p.dq, p.dqs, s);
    }
    if (const char* e = launch(p, DKV, b, s)) return e;
    if (b.n_split > 1 && p.Lk > 0) {
        const float* pv = p.part + (int64_t)b.n_split * p.B * p.Lk * p.Hkv * p.D;
        if (p.dtype == 1) {
            launch_sum<bf16>(p.part, b.n_split, p.B, p.Lk, p.Hkv, p.D, p.dk, p.dks, s);
            launch_sum<bf16>(pv, b.n_split, p.B, p.Lk, p.Hkv, p.D, p.dv, p.dvs, s);
        } else {
            launch_sum<float>(p.part, b.n_split, p.B, p.Lk, p.Hkv, p.D, p.dk, p.dks, s);
            launch_sum<float>(pv, b.n_split, p.B, p.Lk, p.Hkv, p.D, p.dv, p.dvs, s);
        }
    }
    return nullptr;
}

}  // namespace op
}  // namespace tb
