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
template <typename T, int ROWS, int COLS, int NT, bool GATED, bool NARROW>
struct Tile {
    static constexpr int NP = Planes<T>::N, CH = COLS / 8, PT = ROWS * CH / NT, LD = COLS + LDS_PAD;
    static_assert(NT % CH == 0 && ROWS * CH % NT == 0, "a thread's chunks are whole and share their columns");
    Held<T> r[PT];
    Held<T> gate[GATED ? PT : 1];
    uint8_t ok[PT];
    int rows, col_left, shift;
    // rows row0 .. (row0 < row_end) of a [., ld] matrix up to row_end, columns col0 .. (col0 < col_end) up to col_end; what lies outside, or in an
    // invalid row, becomes zero
    __device__ __forceinline__ void load(const T* base, int64_t ld, int64_t row0, int64_t row_end, int col0, int col_end, const Valid& valid, const T* act, int tid) {
        const int col = col0 + (tid % CH) * 8, cc = NARROW ? col < col_end ? col : col0 : chunk_start(col, col_end);
#pragma unroll
        for (int c = 0; c < PT; ++c) {
            const int64_t row = row0 + (tid + c * NT) / CH, rc = row < row_end ? row : row_end - 1;
            if constexpr (NARROW)
                r[c].load_narrow(base + rc * ld + cc, col_end - cc);
            else
                r[c].load(base + rc * ld + cc);
            if constexpr (GATED) {
                if constexpr (NARROW)
                    gate[c].load_narrow(act + rc * ld + cc, col_end - cc);
                else
                    gate[c].load(act + rc * ld + cc);
            }
            ok[c] = valid[rc];
        }
        rows = row_end - row0 < ROWS ? (int)(row_end - row0) : ROWS;
        col_left = col_end - col;
        shift = col - cc;
    }
    // the ends of rows, the masks and the activation's gradient, where the loads are waited for
    __device__ __forceinline__ void settle(bool ragged, int tid) {
        if (!NARROW && ragged) {
#pragma unroll
            for (int c = 0; c < PT; ++c) {
                r[c].fit(shift);
                if constexpr (GATED) gate[c].fit(shift);
            }
        }
        if constexpr (GATED) {
#pragma unroll
            for (int c = 0; c < PT; ++c)
#pragma unroll
                for (int j = 0; j < 8; ++j)
                    if (!(gate[c].get(j) > 0.f)) r[c].drop(j);
        }
#pragma unroll
        for (int c = 0; c < PT; ++c) r[c].keep(ok[c] && (tid + c * NT) / CH < rows && col_left > 0);
    }
    __device__ __forceinline__ void store(bf16* lds, int tid) const {
#pragma unroll
        for (int c = 0; c < PT; ++c) {
            const int idx = tid + c * NT;
            bf16x8 pl[NP];
            r[c].planes(pl);
#pragma unroll
            for (int n = 0; n < NP; ++n) *reinterpret_cast<bf16x8*>(lds + (size_t)n * ROWS * LD + (idx / CH) * LD + (idx % CH) * 8) = pl[n];
        }
    }
    __device__ __forceinline__ void add_columns(float (&s)[8]) const {
#pragma unroll
        for (int c = 0; c < PT; ++c)
#pragma unroll
            for (int j = 0; j < 8; ++j) s[j] += r[c].get(j);
    }
};

// GATED: with the activation's gradient.  NARROW: an operand's rows have fewer than 8 elements.
template <typename T, Kind KIND, bool GATED, int TR, int TC, int WR, int WC, int KB, bool NARROW>
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
    const T* act = GATED ? (const T*)p.act : nullptr;
    const int64_t lda = p.K, ldb = KIND == FWD ? p.K : p.N;

    Tile<T, AR, AC, NT, false, NARROW> ta;
    Tile<T, BR, BC, NT, GATED, NARROW> tb;
    int64_t k0 = (int64_t)split * p.split_len;
    const int64_t kend = KIND == DW ? (k0 + p.split_len < Kn ? k0 + p.split_len : Kn) : Kn;
    const bool ragged_a = lda % 8 != 0, ragged_b = ldb % 8 != 0;
    const Valid rows_valid(p.row_valid, 0), all(nullptr, 0);
    auto load = [&](int64_t k) {
        if constexpr (AT)
            ta.load(A, lda, k, kend, r0, R, KIND == DW ? rows_valid : all, nullptr, tid);
        else
            ta.load(A, lda, r0, R, (int)k, (int)kend, all, nullptr, tid);
        if constexpr (BT)
            tb.load(B, ldb, k, kend, (int)c0, (int)Cn, rows_valid, act, tid);
        else
            tb.load(B, ldb, c0, Cn, (int)k, (int)kend, rows_valid, act, tid);
    };
    f32x4 acc[MC][MR];
#pragma unroll
    for (int c = 0; c < MC; ++c)
#pragma unroll
        for (int r = 0; r < MR; ++r) acc[c][r] = (f32x4){0.f, 0.f, 0.f, 0.f};
    float sums[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
    if (k0 < kend) load(k0);
    for (; k0 < kend; k0 += KB) {
        ta.settle(ragged_a, tid);
        tb.settle(ragged_b, tid);
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
                    store4(p.part + split * ((int64_t)p.N * p.K + p.N) + at, n, v);
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
                        p.part[split * ((int64_t)p.N * p.K + p.N) + (int64_t)p.N * p.K + c0 + c] = s;
                    else
                        ((T*)p.db)[c0 + c] = (T)s;
                }
        }
    }
}

// [dW, db][i] = sum over the splits of part[split][N K + N], always in the same order: 16 groups of 4 elements x 16 lanes over the splits
template <typename T>
__global__ __launch_bounds__(256) void k_linear_sum(const float* part, int n_split, int64_t n_w, int n_b, T* dw, T* db) {
    __shared__ __attribute__((aligned(16))) f32x4 red[16][17];
    const int tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
    const int64_t n = n_w + n_b, i = ((int64_t)blockIdx.x * 16 + tx) * 4;
    f32x4 s = {0.f, 0.f, 0.f, 0.f};
    if (i + 4 <= n) {
        for (int k = ty; k < n_split; k += 16) {
            f32x4 v;
            __builtin_memcpy(&v, part + k * n + i, 16);
            s += v;
        }
    } else {
        for (int k = ty; k < n_split; k += 16)
#pragma unroll
            for (int e = 0; e < 4; ++e)
                if (i + e < n) s[e] += part[k * n + i + e];
    }
    red[ty][tx] = s;
    __syncthreads();
    if (ty) return;
#pragma unroll
    for (int k = 1; k < 16; ++k) s += red[k][tx];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        if (i + e < n_w) {
            if (dw) dw[i + e] = (T)s[e];
        } else if (i + e < n && db) {
            db[i + e - n_w] = (T)s[e];
        }
    }
}

struct Shape {
    void (*kernel)(LinearP);
    int tr, tc, kb, threads;
};
template <typename T, Kind KIND, bool GATED, int TR, int TC, int WR, int WC, bool NARROW>
Shape shape() {
    constexpr int KB = sizeof(T) == 2 ? 64 : 32;
    return {k_linear<T, KIND, GATED, TR, TC, WR, WC, KB, NARROW>, TR, TC, KB, 64 * WR * WC};
}
template <typename T, Kind KIND, bool GATED>
Shape choose(const LinearP& p, int64_t r, int64_t c) {
    if (p.K < 8 || (KIND != FWD && p.N < 8)) return shape<T, KIND, GATED, 64, 64, 2, 2, true>();
    // 128 x 128 tiles feed the matrix cores best; below one such tile per CU the smaller ones spread the work
    if (KIND == DW ? r > 64 || c > 64 : (r + 127) / 128 * ((c + 127) / 128) >= 256) return shape<T, KIND, GATED, 128, 128, 2, 2, false>();
    return shape<T, KIND, GATED, 64, 64, 2, 2, false>();
}
template <typename T, Kind KIND>
Shape choose(const LinearP& p, int64_t r, int64_t c) {
    if constexpr (KIND != FWD)
        if (p.act) return choose<T, KIND, true>(p, r, c);
    return choose<T, KIND, false>(p, r, c);
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
    r.s = p.dtype == 1 ? choose<bf16, KIND>(p, R, C) : choose<float, KIND>(p, R, C);
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
void launch_sum(const LinearP& p, int n_split, hipStream_t s) {
    const int64_t n = (int64_t)p.N * p.K;
    k_linear_sum<T><<<dim3((unsigned)((n + p.N + 63) / 64)), dim3(256), 0, s>>>(p.part, n_split, n, p.N, (T*)p.dw, (T*)p.db);
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
        if (p.dtype == 1)
            launch_sum<bf16>(p, r.p.n_split, s);
        else
            launch_sum<float>(p, r.p.n_split, s);
    }
    return nullptr;
}

}  // namespace op
}  // namespace tb
