// Linear for training: z = x W^T + b, a = relu(z) or z, 0 in invalid rows, y = a + residual; and its backward products
//   dz = dy [a > 0] [row valid],  dx = dz W,  dW = dz^T x,  db = sum over rows of dz.
// One tiled product serves all three: OUT[c][r] = sum_k A(r, k) B(c, k).  The accumulators hold four consecutive r of one column c, so with
// r along the output's rows in memory every lane stores 8 or 16 bytes.
//   forward  r = output feature, c = row of x:   A = W, B = x, both with k along memory
//   dx       r = input feature,  c = row of dy:  A = W with k across memory (read from LDS through the transposing read), B = dz
//   dW       r = input feature,  c = output feature, k = the rows of the batch: both across memory
// The activation's gradient and the row mask are applied to dy while a tile goes to LDS: dz is never stored.  db is the column sum of those
// tiles, taken by the workgroups of the first r tile.  dW's long contraction is split over workgroups; their fp32 parts are added up in
// split order by a second kernel: no atomics, the same bits every run.
#include "tb_ops.hpp"

#include "tb_ops_host.hpp"

namespace tb {
namespace op {

namespace {

enum Kind { FWD, DX, DW };

// A tile of ROWS x COLS elements (a multiple of 8 columns) between global memory and LDS
template <typename T, int ROWS, int COLS, int NT, bool GATED>
struct Tile {
    static constexpr int NP = Planes<T>::N, CH = COLS / 8, PT = (ROWS * CH + NT - 1) / NT, LD = COLS + LDS_PAD;
    static_assert(NT % CH == 0, "a thread's chunks share their columns");
    Held<T> r[PT];
    Held<T> gate[GATED ? PT : 1];
    // rows row0 .. of a [., ld] matrix up to row_end, columns col0 .. up to col_end; what lies outside, or in an invalid row, is zero
    __device__ __forceinline__ void load(const T* base, int64_t ld, int64_t row0, int64_t row_end, int col0, int col_end, const uint8_t* valid, const T* act, int tid) {
#pragma unroll
        for (int c = 0; c < PT; ++c) {
            const int idx = tid + c * NT, col = col0 + (idx % CH) * 8;
            const int64_t row = row0 + idx / CH;
            r[c].zero();
            if constexpr (GATED) gate[c].zero();
            if (idx < ROWS * CH && row < row_end && col < col_end) {
                r[c].load(base + row * ld + col, col_end - col);
                if constexpr (GATED)
                    if (act) gate[c].load(act + row * ld + col, col_end - col);
                if (valid && !valid[row]) r[c].zero();
            }
        }
    }
    __device__ __forceinline__ void apply_gate() {
        if constexpr (GATED) {
#pragma unroll
            for (int c = 0; c < PT; ++c)
#pragma unroll
                for (int j = 0; j < 8; ++j)
                    if (!(gate[c].get(j) > 0.f)) r[c].set(j, 0.f);
        }
    }
    __device__ __forceinline__ void store(bf16* lds, int tid) const {
#pragma unroll
        for (int c = 0; c < PT; ++c) {
            const int idx = tid + c * NT;
            if (ROWS * CH % NT == 0 || idx < ROWS * CH) {
                bf16x8 pl[NP];
                r[c].planes(pl);
#pragma unroll
                for (int n = 0; n < NP; ++n) *reinterpret_cast<bf16x8*>(lds + (size_t)n * ROWS * LD + (idx / CH) * LD + (idx % CH) * 8) = pl[n];
            }
        }
    }
    __device__ __forceinline__ void add_columns(float (&s)[8]) const {
#pragma unroll
        for (int c = 0; c < PT; ++c)
#pragma unroll
            for (int j = 0; j < 8; ++j) s[j] += r[c].get(j);
    }
};

template <typename T, Kind KIND, int TR, int TC, int WR, int WC, int KB>
__global__ __launch_bounds__(64 * WR * WC) void k_linear(const LinearP p) {
    constexpr int NP = Planes<T>::N, NT = 64 * WR * WC, MR = TR / WR / 16, MC = TC / WC / 16;
    constexpr bool AT = KIND != FWD, BT = KIND == DW;  // contraction across memory
    constexpr int AR = AT ? KB : TR, AC = AT ? TR : KB, BR = BT ? KB : TC, BC = BT ? TC : KB, LDA = AC + LDS_PAD, LDB = BC + LDS_PAD;
    __shared__ __attribute__((aligned(16))) bf16 la[NP * AR * LDA];
    __shared__ __attribute__((aligned(16))) bf16 lb[NP * BR * LDB];
    // tiles in XCD order: workgroups go to the eight XCDs round robin; each XCD takes a contiguous part of the tile list, the r tiles of one
    // column tile next to each other, so that its L2 reads the column operand once
    const int64_t total = (int64_t)p.n_rt * p.n_ct * p.n_split, per = (total + 7) / 8, t = (int64_t)(blockIdx.x & 7u) * per + (blockIdx.x >> 3);
    if ((int64_t)(blockIdx.x >> 3) >= per || t >= total) return;
    const int rt = (int)(t % p.n_rt);
    const int64_t ct = t / p.n_rt % p.n_ct;
    const int split = (int)(t / p.n_rt / p.n_ct);
    const int r0 = rt * TR;
    const int64_t c0 = ct * TC;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, i16 = lane & 15, g = lane >> 4;
    const int wr = (wave % WR) * (TR / WR), wc = (wave / WR) * (TC / WC);
    const int R = KIND == FWD ? p.N : p.K;                                   // extent of r
    const int64_t Cn = KIND == DW ? p.N : p.M;                               // extent of c
    const int64_t Kn = KIND == FWD ? p.K : KIND == DX ? p.N : p.M;           // extent of the contraction
    const T* A = KIND == DW ? (const T*)p.x : (const T*)p.weight;
    const T* B = KIND == FWD ? (const T*)p.x : (const T*)p.d_out;
    const T* act = KIND == FWD ? nullptr : (const T*)p.act;
    const int64_t lda = p.K, ldb = KIND == FWD ? p.K : p.N;

    Tile<T, AR, AC, NT, false> ta;
    Tile<T, BR, BC, NT, KIND != FWD> tb;
    int64_t k0 = (int64_t)split * p.split_len;
    const int64_t kend = KIND == DW ? (k0 + p.split_len < Kn ? k0 + p.split_len : Kn) : Kn;
    auto load = [&](int64_t k) {
        if constexpr (AT)
            ta.load(A, lda, k, kend, r0, R, KIND == DW ? p.row_valid : nullptr, nullptr, tid);
        else
            ta.load(A, lda, r0, R, (int)k, (int)kend, nullptr, nullptr, tid);
        if constexpr (BT)
            tb.load(B, ldb, k, kend, (int)c0, (int)Cn, p.row_valid, act, tid);
        else
            tb.load(B, ldb, c0, Cn, (int)k, (int)kend, p.row_valid, act, tid);
    };
    f32x4 acc[MC][MR];
#pragma unroll
    for (int c = 0; c < MC; ++c)
#pragma unroll
        for (int r = 0; r < MR; ++r) acc[c][r] = (f32x4){0.f, 0.f, 0.f, 0.f};
    float sums[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
    if (k0 < kend) load(k0);
    for (; k0 < kend; k0 += KB) {
        if (act) tb.apply_gate();
        if (KIND == DW && rt == 0) tb.add_columns(sums);
        __syncthreads();
        ta.store(la, tid);
        tb.store(lb, tid);
        __syncthreads();
        if (k0 + KB < kend) load(k0 + KB);
#pragma unroll
        for (int kk = 0; kk < KB; kk += 32) {
            Frag<NP> fa[MR];
#pragma unroll
            for (int r = 0; r < MR; ++r) {
                if constexpr (AT)
                    frag_cols<NP, LDA>(la, (size_t)AR * LDA, kk + 8 * g, kk + 8 * g + 4, wr + r * 16, lane, fa[r]);
                else
                    frag_rows<NP, LDA>(la, (size_t)AR * LDA, wr + r * 16, kk, lane, fa[r]);
            }
#pragma unroll
            for (int c = 0; c < MC; ++c) {
                Frag<NP> fb;
                if constexpr (BT)
                    frag_cols<NP, LDB>(lb, (size_t)BR * LDB, kk + 8 * g, kk + 8 * g + 4, wc + c * 16, lane, fb);
                else
                    frag_rows<NP, LDB>(lb, (size_t)BR * LDB, wc + c * 16, kk, lane, fb);
#pragma unroll
                for (int r = 0; r < MR; ++r) acc[c][r] = mma<NP>(fa[r], fb, acc[c][r]);
            }
        }
    }
#pragma unroll
    for (int c = 0; c < MC; ++c) {
        const int64_t col = c0 + wc + c * 16 + i16;
        if (col >= Cn) continue;
#pragma unroll
        for (int r = 0; r < MR; ++r) {
            const int row = r0 + wr + r * 16 + 4 * g, n = R - row;
            if (n <= 0) continue;
            f32x4 v = acc[c][r];
            const int64_t at = col * R + row;
            if constexpr (KIND == FWD) {
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    if (p.bias && e < n) v[e] += (float)((const T*)p.bias)[row + e];
                    if (p.relu) v[e] = v[e] < 0.f ? 0.f : v[e];  // (a NaN stays)
                }
                if (p.row_valid && !p.row_valid[col]) v = (f32x4){0.f, 0.f, 0.f, 0.f};
                if (p.act_out) store4((T*)p.act_out + at, n, v);
                if (p.residual)
#pragma unroll
                    for (int e = 0; e < 4; ++e)
                        if (e < n) v[e] += (float)((const T*)p.residual)[at + e];
                store4((T*)p.y + at, n, v);
            } else if constexpr (KIND == DX) {
                store4((T*)p.dx + at, n, v);
            } else {
                if (p.n_split > 1)
                    store4(p.part + (int64_t)split * p.N * p.K + at, n, v);
                else if (p.dw)
                    store4((T*)p.dw + at, n, v);
            }
        }
    }
    if constexpr (KIND == DW) {
        if (rt == 0 && p.db) {  // (workgroup-uniform) the threads of one chunk of columns add up, in thread order
            constexpr int CH = TC / 8, RT = NT / CH;
            static_assert((size_t)RT * TC * 4 <= sizeof(la) + sizeof(lb) || RT * TC * 4 <= sizeof(la), "the column sums fit the A tile");
            float* red = reinterpret_cast<float*>(la);
            __syncthreads();
#pragma unroll
            for (int j = 0; j < 8; ++j) red[(tid / CH) * TC + (tid % CH) * 8 + j] = sums[j];
            __syncthreads();
            for (int c = tid; c < TC; c += NT)
                if (c0 + c < p.N) {
                    float s = 0.f;
                    for (int k = 0; k < RT; ++k) s += red[k * TC + c];
                    if (p.n_split > 1)
                        p.part[(int64_t)p.n_split * p.N * p.K + (int64_t)split * p.N + c0 + c] = s;
                    else
                        ((T*)p.db)[c0 + c] = (T)s;
                }
        }
    }
}

// dst[i] = sum over the splits, in split order
template <typename T>
__global__ __launch_bounds__(256) void k_linear_sum(const float* part, int n_split, int64_t n, T* dst) {
    const int64_t i = ((int64_t)blockIdx.x * 256 + threadIdx.x) * 4;
    if (i >= n) return;
    f32x4 s = {0.f, 0.f, 0.f, 0.f};
    const int m = n - i < 4 ? (int)(n - i) : 4;
    for (int k = 0; k < n_split; ++k) {
        const float* src = part + k * n + i;
        if (m == 4) {
            f32x4 v;
            __builtin_memcpy(&v, src, 16);
            s += v;
        } else {
#pragma unroll
            for (int e = 0; e < 4; ++e)
                if (e < m) s[e] += src[e];
        }
    }
    store4(dst + i, m, s);
}

struct Shape {
    void (*kernel)(LinearP);
    int tr, tc, kb, threads;
};
template <typename T, Kind KIND, int TR, int TC, int WR, int WC, int KB>
Shape shape() {
    return {k_linear<T, KIND, TR, TC, WR, WC, KB>, TR, TC, KB, 64 * WR * WC};
}
template <typename T, Kind KIND>
Shape choose(int64_t r, int64_t c) {
    constexpr int KB = sizeof(T) == 2 ? 64 : 32;
    // 128 x 128 tiles feed the matrix cores best; below one such tile per CU the smaller ones spread the work
    if (KIND == DW ? r > 64 || c > 64 : (r + 127) / 128 * ((c + 127) / 128) >= 256) return shape<T, KIND, 128, 128, 2, 2, KB>();
    return shape<T, KIND, 64, 64, 2, 2, KB>();
}

struct Plan {
    Shape s;
    LinearP p;
    int64_t blocks;
};
template <Kind KIND>
Plan plan(const LinearP& p) {
    Plan r;
    r.p = p;
    const int64_t R = KIND == FWD ? p.N : p.K, C = KIND == DW ? p.N : p.M;
    r.s = p.dtype == 1 ? choose<bf16, KIND>(R, C) : choose<float, KIND>(R, C);
    r.p.n_rt = (int)((R + r.s.tr - 1) / r.s.tr);
    r.p.n_ct = (C + r.s.tc - 1) / r.s.tc;
    r.p.n_split = 1;
    r.p.split_len = 0;
    if (KIND == DW) {  // about two workgroups per CU; a part keeps at least four tiles of the contraction
        const int64_t tiles = (p.M + r.s.kb - 1) / r.s.kb, base = (int64_t)r.p.n_rt * r.p.n_ct;
        int64_t n = 512 / (base > 0 ? base : 1);
        if (n > tiles / 4) n = tiles / 4;
        if (n < 1) n = 1;
        r.p.split_len = (tiles + n - 1) / n * r.s.kb;
        r.p.n_split = r.p.split_len > 0 ? (int)((p.M + r.p.split_len - 1) / r.p.split_len) : 1;
        if (r.p.n_split < 1) r.p.n_split = 1;
    }
    r.blocks = ((int64_t)r.p.n_rt * r.p.n_ct * r.p.n_split + 7) / 8 * 8;
    return r;
}

const char* launch(const Plan& r, hipStream_t s) {
    if (r.blocks <= 0) return nullptr;
    if (r.blocks > 0x7fffffff) return "too many workgroups (rows x features / tile > 2^31)";
    r.s.kernel<<<dim3((unsigned)r.blocks), dim3(r.s.threads), 0, s>>>(r.p);
    return nullptr;
}

template <typename T>
void launch_sum(const float* part, int n_split, int64_t n, void* dst, hipStream_t s) {
    k_linear_sum<T><<<dim3((unsigned)((n + 1023) / 1024)), dim3(256), 0, s>>>(part, n_split, n, (T*)dst);
}

}  // namespace

int64_t linear_workspace(const LinearP& p) {
    const int n = plan<DW>(p).p.n_split;
    return n > 1 ? 4 * (int64_t)n * ((int64_t)p.N * p.K + p.N) : 0;
}

const char* run_linear(const LinearP& p, hipStream_t s) { return launch(plan<FWD>(p), s); }

const char* run_linear_backward(LinearP p, float* ws, hipStream_t s) {
    if (p.dx)
        if (const char* e = launch(plan<DX>(p), s)) return e;
    if (!p.dw && !p.db) return nullptr;
    p.part = ws;
    const Plan r = plan<DW>(p);
    if (const char* e = launch(r, s)) return e;
    if (r.p.n_split > 1) {
        const int64_t n = (int64_t)p.N * p.K;
        const float* pb = ws + r.p.n_split * n;
        if (p.dtype == 1) {
            if (p.dw) launch_sum<bf16>(ws, r.p.n_split, n, p.dw, s);
            if (p.db) launch_sum<bf16>(pb, r.p.n_split, p.N, p.db, s);
        } else {
            if (p.dw) launch_sum<float>(ws, r.p.n_split, n, p.dw, s);
            if (p.db) launch_sum<float>(pb, r.p.n_split, p.N, p.db, s);
        }
    }
    return nullptr;
}

}  // namespace op
}  // namespace tb
