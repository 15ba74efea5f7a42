// diff_attention.hip — differential attention, forward and backward, on the matrix cores.
//
//   S_j = Q_j K_j^T / sqrt(d) + key mask,  P_j = softmax(S_j)  (j = 1, 2: the two d-wide halves of a head's 2 d query / key columns)
//   o = dropout(P_1 - lambda_h P_2) V,     lambda_h = exp(lq1 . lk1) - exp(lq2 . lk2) + lambda_init
//   y = (1 - lambda_init) w . o / sqrt(mean(o^2) + eps)  per head (w == NULL: y = o)
//
// A head is W = 2 d columns of the q, k, v and y rows: with d = 32 the 64 columns of an ordinary head, with d = 64 two of them.
//
// Orientation: scores are formed transposed (S^T = K Q^T, 32 x 32 x 16 MFMA), so that a lane owns one query (lane & 31) and holds 16 of
// its 32 keys in registers, the other 16 sitting in lane ^ 32: softmax runs over registers plus one swap between the halves of the wave,
// and the registers are, as they stand, the B operand of O^T = V^T P^T (the k order within a step is free as long as V's transposed
// reads follow it).  The backward pass of K and V needs the sums over queries, so there a lane owns one key.
//
// One pass over the keys with running maximum and sum of BOTH maps and one accumulator each: 12 d flops per (query, key) against the
// 8 d of a product with the finished difference, which would need both sums first.
#include "common.cuh"
#include "kernels.h"
#include "../../include/uniter_hip.h"

#include <math.h>

namespace {

typedef __attribute__((ext_vector_type(16))) float f32x16;
typedef __attribute__((ext_vector_type(8))) short s16x8;

constexpr float LOG2E = 1.44269504088896340736f;
constexpr int KT = 64;                   // rows of a staged tile
constexpr int NSTAT = 4;                 // saved per (row, head): max and log2(sum) of both maps, in log2 units

struct DiffArgs {
    const bf16_t *q, *k, *v;
    int64_t lq, lk, lv, bq, bk, bv;      // strides in elements: row, batch
    const float* mask;                   // [B, Lk], row stride lmask, or NULL
    int64_t lmask;
    const int32_t *cu_q, *cu_k;          // packed rows, or NULL
    int64_t tot_q, tot_k;
    const bf16_t *lq1, *lk1, *lq2, *lk2;
    int lam_stride;                      // d: one set of vectors per head; 0: one for all
    float lambda_init;
    const bf16_t* w;
    float eps;
    int B, heads;
    int Lq, Lk;                          // rows per example (packed: the longest)
    float sc;                            // log2(e) / sqrt(d)
    DropoutCfg drop;
    bf16_t* out;                         // forward: rows [.., heads * W]
    int64_t lo, bo;
    float* stats;                        // [B, heads, Lq, NSTAT] or NULL
    float* maps;                         // [row, heads, 2, W]: P_1 V and P_2 V, or NULL
    // backward
    const bf16_t* dout;
    int64_t ldo, bdo;
    bf16_t* dctx;                        // [row, heads * W]: gradient of o
    float* D;                            // [B, heads, Lq, 2]
    bf16_t *dq, *dk, *dv;
    int64_t ldq, ldk, ldv, bdq, bdk, bdv;
    float* part_lam;                     // [heads, chunks]
    float* part_w;                       // [heads, chunks, W]
    int chunks;
};

// ---- LDS tiles: [rows][W] bf16, 16-byte chunk c of row r at c ^ key(r).  The keys spread 8 consecutive rows of one chunk (row
// fragments) and the 4 rows x 2 chunks of a transposed read over different banks.
template <int W>
__device__ __forceinline__ int tile_off(const int r, const int c16) {
    if constexpr (W == 64) return r * 64 + ((c16 ^ (((r >> 1) & 3) << 1)) << 3);
    else return r * 128 + ((c16 ^ ((r & 7) << 1)) << 3);
}
// A / B fragment of a 32-row block: lane (row = lane & 31, half = lane >> 5) reads 8 elements of k step `ks`
template <int W>
__device__ __forceinline__ bf16x8 row_frag(const bf16_t* tile, const int r, const int c16) {
    return *reinterpret_cast<const bf16x8*>(tile + tile_off<W>(r, c16));
}
// transposed fragment: column col0 + (lane & 31), the 8 rows r0 + 4 half + {0..3} and r0 + 8 + 4 half + {0..3}
template <int W>
__device__ __forceinline__ bf16x8 tr_frag(const bf16_t* tile, const int r0, const int col0, const int lane) {
    typedef __attribute__((address_space(3))) s16x4 lds_s16x4;
    const int r = r0 + 4 * (lane >> 5) + ((lane & 15) >> 2);
    const int c4 = (col0 >> 2) + ((lane >> 4) & 1) * 4 + (lane & 3);         // 8-byte chunk
    const s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)(tile + tile_off<W>(r, c4 >> 1) + (c4 & 1) * 4));
    const s16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)(tile + tile_off<W>(r + 8, c4 >> 1) + (c4 & 1) * 4));
    s16x8 v;
    v[0] = lo[0]; v[1] = lo[1]; v[2] = lo[2]; v[3] = lo[3];
    v[4] = hi[0]; v[5] = hi[1]; v[6] = hi[2]; v[7] = hi[3];
    return __builtin_bit_cast(bf16x8, v);
}
__device__ __forceinline__ f32x16 mfma32(const bf16x8 a, const bf16x8 b, const f32x16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
}
__device__ __forceinline__ f32x16 zero16() {
    f32x16 z;
#pragma unroll
    for (int i = 0; i < 16; ++i) z[i] = 0.f;
    return z;
}
// registers 8 kk .. 8 kk + 7 of an accumulator as the operand of k step kk
__device__ __forceinline__ bf16x8 pack_step(const f32x16& s, const int kk) {
    u32x4 w;
#pragma unroll
    for (int i = 0; i < 4; ++i) w[i] = pack_bf16x2(s[8 * kk + 2 * i], s[8 * kk + 2 * i + 1]);
    return __builtin_bit_cast(bf16x8, w);
}
// the value of lane ^ 32
__device__ __forceinline__ float other_half(const float x) { return __shfl_xor(x, 32, WAVE); }
// row (or column) of an accumulator register: 8 (r / 4) + 4 half + r % 4
__device__ __forceinline__ constexpr int acc_row(const int r) { return 8 * (r >> 2) + (r & 3); }

// A lane holds columns 8 g + 4 half + {0..3}, g = 0..3, of one 32-column block of its row.  The two halves swap a group of every pair,
// so that a lane stores 16 bytes: half 0 the 8 columns of the even group, half 1 those of the odd one.
__device__ __forceinline__ void store_block32(bf16_t* row, const f32x16& v, const int half, const bool valid) {
#pragma unroll
    for (int g = 0; g < 4; g += 2) {
        uint32_t a[2], b[2];
#pragma unroll
        for (int e = 0; e < 2; ++e) {
            a[e] = pack_bf16x2(v[4 * g + 2 * e], v[4 * g + 2 * e + 1]);
            b[e] = pack_bf16x2(v[4 * g + 4 + 2 * e], v[4 * g + 4 + 2 * e + 1]);
        }
        const uint32_t s0 = half ? a[0] : b[0], s1 = half ? a[1] : b[1];
        const uint32_t r0 = (uint32_t)__shfl_xor((int)s0, 32, WAVE), r1 = (uint32_t)__shfl_xor((int)s1, 32, WAVE);
        const u32x4 w = half ? u32x4{r0, r1, b[0], b[1]} : u32x4{a[0], a[1], r0, r1};
        if (valid) out_store16(row + 8 * (g + half), w);
    }
}

// ---- examples: rows [q0, q0 + nq) of q / out and [k0, k0 + nk) of k / v
struct Span { int64_t row; int n; };
__device__ __forceinline__ Span span_of(const int32_t* cu, const int64_t total, const int b, const int L) {
    Span s;
    if (cu == nullptr) { s.row = 0; s.n = L; return s; }
    // (bounds that do not ascend within the rows there are read nothing outside them)
    const int64_t lo = min(max((int64_t)cu[b], (int64_t)0), total), hi = min(max((int64_t)cu[b + 1], lo), total);
    s.row = lo;
    s.n = (int)min(hi - lo, (int64_t)L);
    return s;
}

// additive mask in log2 units; the type's lowest value stays finite (a row of nothing but that is uniform over its keys)
__device__ __forceinline__ float mask_log2(const float m) { return m == -INFINITY ? m : fmaxf(m * LOG2E, -3.4028234663852886e38f); }

// copy KT rows x W columns into a tile; rows from n on, and rows whose mask is -inf (keep(r) false), become zeros: whatever stands
// there, their weight is zero and 0 * NaN must not reach a sum
template <int W, typename Keep>
__device__ __forceinline__ void stage(bf16_t* tile, const bf16_t* src, const int64_t ld, const int r0, const int n, Keep&& keep) {
    for (int e = threadIdx.x; e < KT * (W / 8); e += blockDim.x) {
        const int r = e / (W / 8), c = e % (W / 8);
        u32x4 v = {0u, 0u, 0u, 0u};
        if (r0 + r < n && keep(r)) v = ldg16<false>(src + (int64_t)(r0 + r) * ld + c * 8);
        *reinterpret_cast<u32x4*>(tile + tile_off<W>(r, c)) = v;
    }
}

// mask of the tile's keys (log2 units, -inf behind the end).  All threads of the workgroup call; a barrier follows.
__device__ __forceinline__ void stage_mask(float* mb, const DiffArgs& p, const int b, const int k0, const int nk) {
    if (threadIdx.x < KT) {
        const int key = k0 + (int)threadIdx.x;
        float m = -INFINITY;
        if (key < nk) m = p.mask != nullptr ? mask_log2(p.mask[(int64_t)b * p.lmask + key]) : 0.f;
        mb[threadIdx.x] = m;
    }
}

// lambda of head h (every lane gets it)
template <int D>
__device__ __forceinline__ void lambda_of(const DiffArgs& p, const int h, const int lane, float& e1, float& e2) {
    float a = 0.f, b = 0.f;
    if (lane < D) {
        const int at = h * p.lam_stride + lane;
        a = bf2f(p.lq1[at]) * bf2f(p.lk1[at]);
        b = bf2f(p.lq2[at]) * bf2f(p.lk2[at]);
    }
    e1 = __expf(wave_sum(a));
    e2 = __expf(wave_sum(b));
}

// keep bits of the 16 elements (query of this lane, 32 keys from kb): bit r belongs to register r.  One generator call covers the 8
// registers of a 16-key step that one lane holds: group ((row * ceil(Lk / 16) + key / 16) * 2 + half).
__device__ __forceinline__ uint32_t keep16(const DiffArgs& p, const uint64_t row, const int kb, const int half) {
    const uint64_t n16 = (uint64_t)((p.Lk + 15) >> 4);
    const uint64_t g = (row * n16 + (uint64_t)(kb >> 4)) * 2 + (uint64_t)half;
    return dropout_keep8(p.drop, g) | (dropout_keep8(p.drop, g + 2) << 8);
}

// ------------------------------------------------------------------------------------------------
// forward
// ------------------------------------------------------------------------------------------------
template <int D, bool DROP>
__global__ __launch_bounds__(256) void diff_fwd_kernel(const DiffArgs p, const int nqb) {
    constexpr int W = 2 * D, NS = D / 16, NV = W / 32;
    __shared__ __attribute__((aligned(16))) bf16_t Ks[KT * W];
    __shared__ __attribute__((aligned(16))) bf16_t Vs[KT * W];
    __shared__ __attribute__((aligned(16))) float mb[KT];
    const int bid = xcd_remap((int)blockIdx.x, (int)gridDim.x);
    const int bh = bid / nqb, qb = bid - bh * nqb;
    const int b = bh / p.heads, h = bh - b * p.heads;
    const Span sq = span_of(p.cu_q, p.tot_q, b, p.Lq), sk = span_of(p.cu_k, p.tot_k, b, p.Lk);
    const int lane = threadIdx.x & 63, wid = threadIdx.x >> 6, half = lane >> 5;
    const int nw = (int)blockDim.x >> 6;
    if (qb * nw * 32 >= sq.n) return;
    const int q = (qb * nw + wid) * 32 + (lane & 31);
    const bool live = q < sq.n;
    const bf16_t* Q = p.q + (int64_t)b * p.bq * (p.cu_q == nullptr) + sq.row * p.lq + h * W;
    const bf16_t* K = p.k + (int64_t)b * p.bk * (p.cu_k == nullptr) + sk.row * p.lk + h * W;
    const bf16_t* V = p.v + (int64_t)b * p.bv * (p.cu_k == nullptr) + sk.row * p.lv + h * W;

    bf16x8 qf[2][NS];
#pragma unroll
    for (int j = 0; j < 2; ++j)
#pragma unroll
        for (int s = 0; s < NS; ++s) {
            u32x4 v = {0u, 0u, 0u, 0u};
            if (live) v = ldg16<false>(Q + (int64_t)q * p.lq + j * D + s * 16 + half * 8);
            qf[j][s] = __builtin_bit_cast(bf16x8, v);
        }
    float e1, e2;
    lambda_of<D>(p, h, lane, e1, e2);
    const float lam = e1 - e2 + p.lambda_init;

    f32x16 o[2][NV];
    float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f};
#pragma unroll
    for (int j = 0; j < 2; ++j)
#pragma unroll
        for (int t = 0; t < NV; ++t) o[j][t] = zero16();
    const uint64_t drow = (uint64_t)bh * (uint64_t)p.Lq + (uint64_t)q;

    for (int k0 = 0; k0 < sk.n; k0 += KT) {
        __syncthreads();
        stage_mask(mb, p, b, k0, sk.n);
        __syncthreads();
        stage<W>(Ks, K, p.lk, k0, sk.n, [&](int r) { return mb[r] != -INFINITY; });
        stage<W>(Vs, V, p.lv, k0, sk.n, [&](int r) { return mb[r] != -INFINITY; });
        __syncthreads();
#pragma unroll
        for (int kt = 0; kt < KT / 32; ++kt) {
            uint32_t keep = 0xffffu;
            if constexpr (DROP) keep = keep16(p, drow, k0 + kt * 32, half);
            f32x4 mv[4];
#pragma unroll
            for (int g = 0; g < 4; ++g) mv[g] = *reinterpret_cast<const f32x4*>(mb + kt * 32 + 8 * g + 4 * half);
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                f32x16 s = zero16();
#pragma unroll
                for (int ks = 0; ks < NS; ++ks)
                    s = mfma32(row_frag<W>(Ks, kt * 32 + (lane & 31), (j * D + ks * 16) / 8 + half), qf[j][ks], s);
                float mx = -INFINITY;
#pragma unroll
                for (int r = 0; r < 16; ++r) {
                    s[r] = __builtin_fmaf(s[r], p.sc, mv[r >> 2][r & 3]);
                    mx = fmaxf(mx, s[r]);
                }
                mx = fmaxf(mx, other_half(mx));
                const float mn = fmaxf(m[j], mx);
                const float ms = mn == -INFINITY ? 0.f : mn;                  // (a row that has met no key yet)
                const float alpha = __builtin_amdgcn_exp2f(m[j] - ms);
                m[j] = mn;
                float sum = 0.f;
#pragma unroll
                for (int r = 0; r < 16; ++r) {
                    s[r] = __builtin_amdgcn_exp2f(s[r] - ms);
                    sum += s[r];
                    if constexpr (DROP) s[r] = (keep >> r) & 1u ? s[r] : 0.f;
                }
                l[j] = l[j] * alpha + sum;
#pragma unroll
                for (int t = 0; t < NV; ++t) {
                    o[j][t] *= alpha;
#pragma unroll
                    for (int kk = 0; kk < 2; ++kk)
                        o[j][t] = mfma32(tr_frag<W>(Vs, kt * 32 + kk * 16, t * 32, lane), pack_step(s, kk), o[j][t]);
                }
            }
        }
    }
    const float dscale = DROP ? p.drop.scale : 1.f;
    float inv[2], ll[2];
#pragma unroll
    for (int j = 0; j < 2; ++j) {
        l[j] += other_half(l[j]);
        inv[j] = l[j] > 0.f ? dscale / l[j] : (l[j] == 0.f ? 0.f : l[j]);
        ll[j] = l[j] == 0.f ? INFINITY : __log2f(l[j]);
    }
    const int64_t row = p.cu_q != nullptr ? sq.row + q : (int64_t)b * p.Lq + q;
    if (p.stats != nullptr && live && half == 0) {
        const f32x4 st = {m[0] == -INFINITY ? 0.f : m[0], ll[0], m[1] == -INFINITY ? 0.f : m[1], ll[1]};
        *reinterpret_cast<f32x4*>(p.stats + ((int64_t)bh * p.Lq + q) * NSTAT) = st;
    }
    float ss = 0.f;
#pragma unroll
    for (int t = 0; t < NV; ++t) {
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            o[j][t] *= inv[j];
            if (p.maps != nullptr && live) {
                float* at = p.maps + ((row * p.heads + h) * 2 + j) * W + t * 32 + 4 * half;
#pragma unroll
                for (int g = 0; g < 4; ++g) *reinterpret_cast<f32x4*>(at + 8 * g) = f32x4{o[j][t][4 * g], o[j][t][4 * g + 1], o[j][t][4 * g + 2], o[j][t][4 * g + 3]};
            }
        }
#pragma unroll
        for (int r = 0; r < 16; ++r) {
            o[0][t][r] -= lam * o[1][t][r];
            ss += o[0][t][r] * o[0][t][r];
        }
    }
    if (p.w != nullptr) {
        ss += other_half(ss);
        const float rs = rsqrtf(ss * (1.f / W) + p.eps) * (1.f - p.lambda_init);
#pragma unroll
        for (int t = 0; t < NV; ++t)
#pragma unroll
            for (int r = 0; r < 16; ++r) o[0][t][r] *= rs * bf2f(p.w[t * 32 + acc_row(r) + 4 * half]);
    }
    bf16_t* out = p.out + (int64_t)b * p.bo * (p.cu_q == nullptr) + (sq.row + q) * p.lo + h * W;
#pragma unroll
    for (int t = 0; t < NV; ++t) store_block32(out + t * 32, o[0][t], half, live);
}

// ------------------------------------------------------------------------------------------------
// backward, rows: gradient of o through the sub-normalisation, D_j = dO . (P_j V), and the sums behind dlambda and dw
// ------------------------------------------------------------------------------------------------
// W / 8 lanes per (row, head), 8 columns each; a workgroup takes a chunk of the rows of one (example, head) pair's query rows.
template <int W>
__global__ __launch_bounds__(256) void diff_bwd_rows_kernel(const DiffArgs p, const int rows_per) {
    constexpr int LN = W / 8, RP = 256 / LN;
    __shared__ float sw[RP][W];
    __shared__ float sl[RP];
    const int h = (int)blockIdx.y, lane = threadIdx.x & 63;
    const int c = ((int)threadIdx.x % LN) * 8, ri = (int)threadIdx.x / LN;
    float e1, e2;
    lambda_of<W / 2>(p, h, lane, e1, e2);
    const float lam = e1 - e2 + p.lambda_init, so = 1.f - p.lambda_init;
    float wv[8], aw[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f}, al = 0.f;
    if (p.w != nullptr) unpack8(*reinterpret_cast<const u32x4*>(p.w + c), wv);
    // rows are counted over all examples: (b, q), q < Lq
    const int64_t total = (int64_t)p.B * p.Lq;
    const int64_t r0 = (int64_t)blockIdx.x * rows_per;
    for (int i = ri; i < rows_per; i += RP) {
        const int64_t rr = r0 + i;
        const int b = (int)(rr / p.Lq), q = (int)(rr - (int64_t)b * p.Lq);
        bool ok = rr < total;
        Span sq{0, 0};
        if (ok) { sq = span_of(p.cu_q, p.tot_q, b, p.Lq); ok = q < sq.n; }
        const int64_t row = p.cu_q != nullptr ? sq.row + q : rr;
        float dy[8], o1[8], o2[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) { dy[e] = 0.f; o1[e] = 0.f; o2[e] = 0.f; }
        if (ok) {
            unpack8(*reinterpret_cast<const u32x4*>(p.dout + (int64_t)b * p.bdo * (p.cu_q == nullptr) + (sq.row + q) * p.ldo + h * W + c), dy);
            const f32x4* m = reinterpret_cast<const f32x4*>(p.maps + (row * p.heads + h) * 2 * W + c);
#pragma unroll
            for (int e = 0; e < 8; ++e) { o1[e] = m[e >> 2][e & 3]; o2[e] = m[W / 4 + (e >> 2)][e & 3]; }
        }
        float d[8];
        if (p.w != nullptr) {
            float ss = 0.f, dot = 0.f, o[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                o[e] = o1[e] - lam * o2[e];
                d[e] = so * wv[e] * dy[e];
                ss += o[e] * o[e];
                dot += d[e] * o[e];
            }
#pragma unroll
            for (int s = 1; s < LN; s <<= 1) { ss += __shfl_xor(ss, s, WAVE); dot += __shfl_xor(dot, s, WAVE); }
            const float r = rsqrtf(ss * (1.f / W) + p.eps), cf = r * r * dot * (1.f / W);
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                aw[e] += so * dy[e] * o[e] * r;
                d[e] = r * (d[e] - o[e] * cf);
            }
        } else {
#pragma unroll
            for (int e = 0; e < 8; ++e) d[e] = dy[e];
        }
        // the products that follow take dO as bf16 operands; D and dlambda are formed from the values before that rounding
        float d1 = 0.f, d2 = 0.f;
#pragma unroll
        for (int e = 0; e < 8; ++e) { d1 += d[e] * o1[e]; d2 += d[e] * o2[e]; }
#pragma unroll
        for (int s = 1; s < LN; s <<= 1) { d1 += __shfl_xor(d1, s, WAVE); d2 += __shfl_xor(d2, s, WAVE); }
        if (ok) {
            if (p.dctx != nullptr) *reinterpret_cast<u32x4*>(p.dctx + (row * p.heads + h) * W + c) = pack8(d);
            if (c == 0) {
                float* D = p.D + (((int64_t)b * p.heads + h) * p.Lq + q) * 2;
                D[0] = d1;
                D[1] = d2;
                al -= d2;
            }
        }
    }
#pragma unroll
    for (int e = 0; e < 8; ++e) sw[ri][c + e] = aw[e];
    if (c == 0) sl[ri] = al;
    __syncthreads();
    const int64_t at = (int64_t)h * p.chunks + blockIdx.x;
    if ((int)threadIdx.x < W && p.w != nullptr) {
        float s = 0.f;
        for (int i = 0; i < RP; ++i) s += sw[i][threadIdx.x];
        p.part_w[at * W + threadIdx.x] = s;
    }
    if (threadIdx.x == 0) {
        float s = 0.f;
        for (int i = 0; i < RP; ++i) s += sl[i];
        p.part_lam[at] = s;
    }
}

// ---- sums of the partials -> gradients of the four lambda vectors and of w.  Block 0 .. n_lam - 1: one set of lambda vectors each
// (one per head, or one over all heads); behind them W / 8 blocks of 8 columns of dw.  Summation order is fixed.
struct ParamGrads { bf16_t *lq1, *lk1, *lq2, *lk2, *w; int n_lam, accumulate; };
template <int D>
__global__ __launch_bounds__(256) void diff_bwd_params_kernel(const DiffArgs p, const ParamGrads g) {
    constexpr int W = 2 * D;
    __shared__ float red[256];
    const int tid = (int)threadIdx.x;
    if ((int)blockIdx.x < g.n_lam) {
        const int h = (int)blockIdx.x;
        const int64_t n = (int64_t)p.chunks * (g.n_lam == 1 ? p.heads : 1);
        const float* src = p.part_lam + (g.n_lam == 1 ? 0 : (int64_t)h * p.chunks);
        float s = 0.f;
        for (int64_t i = tid; i < n; i += 256) s += src[i];
        red[tid] = s;
        __syncthreads();
        for (int k = 128; k > 0; k >>= 1) {
            if (tid < k) red[tid] += red[tid + k];
            __syncthreads();
        }
        if (tid < 64) {
            float e1, e2;
            lambda_of<D>(p, h, tid, e1, e2);
            const float d1 = red[0] * e1, d2 = -red[0] * e2;
            if (tid < D) {
                const int at = h * p.lam_stride + tid;
                auto put = [&](bf16_t* dst, float v) { if (dst != nullptr) dst[at] = f2bf(g.accumulate ? bf2f(dst[at]) + v : v); };
                put(g.lq1, d1 * bf2f(p.lk1[at]));
                put(g.lk1, d1 * bf2f(p.lq1[at]));
                put(g.lq2, d2 * bf2f(p.lk2[at]));
                put(g.lk2, d2 * bf2f(p.lq2[at]));
            }
        }
        return;
    }
    const int c = ((int)blockIdx.x - g.n_lam) * 8 + (tid & 7);
    float s = 0.f;
    for (int64_t i = tid >> 3; i < (int64_t)p.heads * p.chunks; i += 32) s += p.part_w[i * W + c];
    red[tid] = s;
    __syncthreads();
    for (int k = 128; k >= 8; k >>= 1) {
        if (tid < k) red[tid] += red[tid + k];
        __syncthreads();
    }
    if (tid < 8) g.w[c] = f2bf(g.accumulate ? bf2f(g.w[c]) + red[tid] : red[tid]);
}

// ------------------------------------------------------------------------------------------------
// backward, queries: dQ_j = sum_k dS_j K_j,  dS_1 = P_1 (G - D_1) / sqrt(d),  dS_2 = -lambda P_2 (G - D_2) / sqrt(d),  G = dropout(dO V^T)
// ------------------------------------------------------------------------------------------------
template <int D, bool DROP>
__global__ __launch_bounds__(256) void diff_bwd_dq_kernel(const DiffArgs p, const int nqb) {
    constexpr int W = 2 * D, NS = D / 16, ND = D / 32;
    __shared__ __attribute__((aligned(16))) bf16_t Ks[KT * W];
    __shared__ __attribute__((aligned(16))) bf16_t Vs[KT * W];
    __shared__ __attribute__((aligned(16))) float mb[KT];
    const int bid = xcd_remap((int)blockIdx.x, (int)gridDim.x);
    const int bh = bid / nqb, qb = bid - bh * nqb;
    const int b = bh / p.heads, h = bh - b * p.heads;
    const Span sq = span_of(p.cu_q, p.tot_q, b, p.Lq), sk = span_of(p.cu_k, p.tot_k, b, p.Lk);
    const int lane = threadIdx.x & 63, wid = threadIdx.x >> 6, half = lane >> 5;
    const int nw = (int)blockDim.x >> 6;
    if (qb * nw * 32 >= sq.n) return;
    const int q = (qb * nw + wid) * 32 + (lane & 31);
    const bool live = q < sq.n;
    const bf16_t* Q = p.q + (int64_t)b * p.bq * (p.cu_q == nullptr) + sq.row * p.lq + h * W;
    const bf16_t* K = p.k + (int64_t)b * p.bk * (p.cu_k == nullptr) + sk.row * p.lk + h * W;
    const bf16_t* V = p.v + (int64_t)b * p.bv * (p.cu_k == nullptr) + sk.row * p.lv + h * W;
    const bool own = p.dctx != nullptr;
    const bf16_t* dO = own ? p.dctx + ((p.cu_q != nullptr ? sq.row : (int64_t)b * p.Lq) * p.heads + h) * W
                           : p.dout + (int64_t)b * p.bdo * (p.cu_q == nullptr) + sq.row * p.ldo + h * W;
    const int64_t ldO = own ? (int64_t)p.heads * W : p.ldo;

    bf16x8 qf[2][NS], gf[W / 16];
#pragma unroll
    for (int s = 0; s < W / 16; ++s) {
        u32x4 v = {0u, 0u, 0u, 0u}, d = {0u, 0u, 0u, 0u};
        if (live) {
            v = ldg16<false>(Q + (int64_t)q * p.lq + s * 16 + half * 8);
            d = ldg16<false>(dO + (int64_t)q * ldO + s * 16 + half * 8);
        }
        qf[s / NS][s % NS] = __builtin_bit_cast(bf16x8, v);
        gf[s] = __builtin_bit_cast(bf16x8, d);
    }
    float m[2] = {0.f, 0.f}, ll[2] = {INFINITY, INFINITY}, Dq[2] = {0.f, 0.f};
    if (live) {
        const f32x4 st = *reinterpret_cast<const f32x4*>(p.stats + ((int64_t)bh * p.Lq + q) * NSTAT);
        m[0] = st[0]; ll[0] = st[1]; m[1] = st[2]; ll[1] = st[3];
        Dq[0] = p.D[((int64_t)bh * p.Lq + q) * 2];
        Dq[1] = p.D[((int64_t)bh * p.Lq + q) * 2 + 1];
    }
    float e1, e2;
    lambda_of<D>(p, h, lane, e1, e2);
    const float lam = e1 - e2 + p.lambda_init;
    const uint64_t drow = (uint64_t)bh * (uint64_t)p.Lq + (uint64_t)q;
    const float dscale = DROP ? p.drop.scale : 1.f;

    f32x16 dq[2][ND];
#pragma unroll
    for (int j = 0; j < 2; ++j)
#pragma unroll
        for (int t = 0; t < ND; ++t) dq[j][t] = zero16();

    for (int k0 = 0; k0 < sk.n; k0 += KT) {
        __syncthreads();
        stage_mask(mb, p, b, k0, sk.n);
        __syncthreads();
        stage<W>(Ks, K, p.lk, k0, sk.n, [&](int r) { return mb[r] != -INFINITY; });
        stage<W>(Vs, V, p.lv, k0, sk.n, [&](int r) { return mb[r] != -INFINITY; });
        __syncthreads();
#pragma unroll
        for (int kt = 0; kt < KT / 32; ++kt) {
            f32x16 g = zero16();
#pragma unroll
            for (int s = 0; s < W / 16; ++s) g = mfma32(row_frag<W>(Vs, kt * 32 + (lane & 31), 2 * s + half), gf[s], g);
            if constexpr (DROP) {
                const uint32_t keep = keep16(p, drow, k0 + kt * 32, half);
#pragma unroll
                for (int r = 0; r < 16; ++r) g[r] = (keep >> r) & 1u ? g[r] * dscale : 0.f;
            }
            f32x4 mv[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) mv[i] = *reinterpret_cast<const f32x4*>(mb + kt * 32 + 8 * i + 4 * half);
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                f32x16 s = zero16();
#pragma unroll
                for (int ks = 0; ks < NS; ++ks)
                    s = mfma32(row_frag<W>(Ks, kt * 32 + (lane & 31), (j * D + ks * 16) / 8 + half), qf[j][ks], s);
#pragma unroll
                for (int r = 0; r < 16; ++r) {
                    const float pr = __builtin_amdgcn_exp2f((__builtin_fmaf(s[r], p.sc, mv[r >> 2][r & 3]) - m[j]) - ll[j]);
                    s[r] = pr * (g[r] - Dq[j]);
                }
#pragma unroll
                for (int t = 0; t < ND; ++t)
#pragma unroll
                    for (int kk = 0; kk < 2; ++kk)
                        dq[j][t] = mfma32(tr_frag<W>(Ks, kt * 32 + kk * 16, j * D + t * 32, lane), pack_step(s, kk), dq[j][t]);
            }
        }
    }
    const float z = p.sc * (1.f / LOG2E);
    bf16_t* dst = p.dq + (int64_t)b * p.bdq * (p.cu_q == nullptr) + (sq.row + q) * p.ldq + h * W;
#pragma unroll
    for (int j = 0; j < 2; ++j)
#pragma unroll
        for (int t = 0; t < ND; ++t) {
            dq[j][t] *= j == 0 ? z : -lam * z;
            store_block32(dst + j * D + t * 32, dq[j][t], half, live);
        }
}

// ------------------------------------------------------------------------------------------------
// backward, keys: dV = sum_q A dO with A = dropout(P_1 - lambda P_2);  dK_j = sum_q dS_j Q_j
// ------------------------------------------------------------------------------------------------
template <int D, bool DROP>
__global__ __launch_bounds__(256) void diff_bwd_dkv_kernel(const DiffArgs p, const int nkb) {
    constexpr int W = 2 * D, NS = D / 16, ND = D / 32, NV = W / 32;
    __shared__ __attribute__((aligned(16))) bf16_t Qs[KT * W];
    __shared__ __attribute__((aligned(16))) bf16_t Os[KT * W];
    __shared__ __attribute__((aligned(16))) float st[6][KT];      // m1, log2 l1, m2, log2 l2, D1, D2
    const int bid = xcd_remap((int)blockIdx.x, (int)gridDim.x);
    const int bh = bid / nkb, kb = bid - bh * nkb;
    const int b = bh / p.heads, h = bh - b * p.heads;
    const Span sq = span_of(p.cu_q, p.tot_q, b, p.Lq), sk = span_of(p.cu_k, p.tot_k, b, p.Lk);
    const int lane = threadIdx.x & 63, wid = threadIdx.x >> 6, half = lane >> 5;
    const int nw = (int)blockDim.x >> 6;
    if (kb * nw * 32 >= sk.n) return;
    const int kbase = (kb * nw + wid) * 32, key = kbase + (lane & 31);
    const bool live = key < sk.n;
    const bf16_t* Q = p.q + (int64_t)b * p.bq * (p.cu_q == nullptr) + sq.row * p.lq + h * W;
    const bf16_t* K = p.k + (int64_t)b * p.bk * (p.cu_k == nullptr) + sk.row * p.lk + h * W;
    const bf16_t* V = p.v + (int64_t)b * p.bv * (p.cu_k == nullptr) + sk.row * p.lv + h * W;
    const bool own = p.dctx != nullptr;
    const bf16_t* dO = own ? p.dctx + ((p.cu_q != nullptr ? sq.row : (int64_t)b * p.Lq) * p.heads + h) * W
                           : p.dout + (int64_t)b * p.bdo * (p.cu_q == nullptr) + sq.row * p.ldo + h * W;
    const int64_t ldO = own ? (int64_t)p.heads * W : p.ldo;

    float mk = -INFINITY;
    if (live) mk = p.mask != nullptr ? mask_log2(p.mask[(int64_t)b * p.lmask + key]) : 0.f;
    const bool use = mk != -INFINITY;
    bf16x8 kf[2][NS], vf[W / 16];
#pragma unroll
    for (int s = 0; s < W / 16; ++s) {
        u32x4 a = {0u, 0u, 0u, 0u}, c = {0u, 0u, 0u, 0u};
        if (use) {
            a = ldg16<false>(K + (int64_t)key * p.lk + s * 16 + half * 8);
            c = ldg16<false>(V + (int64_t)key * p.lv + s * 16 + half * 8);
        }
        kf[s / NS][s % NS] = __builtin_bit_cast(bf16x8, a);
        vf[s] = __builtin_bit_cast(bf16x8, c);
    }
    float e1, e2;
    lambda_of<D>(p, h, lane, e1, e2);
    const float lam = e1 - e2 + p.lambda_init;
    const float dscale = DROP ? p.drop.scale : 1.f;

    f32x16 dk[2][ND], dv[NV];
#pragma unroll
    for (int t = 0; t < NV; ++t) dv[t] = zero16();
#pragma unroll
    for (int j = 0; j < 2; ++j)
#pragma unroll
        for (int t = 0; t < ND; ++t) dk[j][t] = zero16();

    for (int q0 = 0; q0 < sq.n; q0 += KT) {
        __syncthreads();
        stage<W>(Qs, Q, p.lq, q0, sq.n, [](int) { return true; });
        stage<W>(Os, dO, ldO, q0, sq.n, [](int) { return true; });
        if (threadIdx.x < KT) {
            const int t = (int)threadIdx.x, q = q0 + t;
            float v[6] = {0.f, INFINITY, 0.f, INFINITY, 0.f, 0.f};           // behind the last query: P = 0
            if (q < sq.n) {
                const f32x4 s4 = *reinterpret_cast<const f32x4*>(p.stats + ((int64_t)bh * p.Lq + q) * NSTAT);
                v[0] = s4[0]; v[1] = s4[1]; v[2] = s4[2]; v[3] = s4[3];
                v[4] = p.D[((int64_t)bh * p.Lq + q) * 2];
                v[5] = p.D[((int64_t)bh * p.Lq + q) * 2 + 1];
            }
#pragma unroll
            for (int i = 0; i < 6; ++i) st[i][t] = v[i];
        }
        __syncthreads();
#pragma unroll
        for (int qt = 0; qt < KT / 32; ++qt) {
            uint32_t keep = 0xffffu;
            if constexpr (DROP) {
                // the bits come out with a query per lane; the ballot of register r is key acc_row(r) + 4 (lane half) over the queries
                const uint64_t drow = (uint64_t)bh * (uint64_t)p.Lq + (uint64_t)(q0 + qt * 32 + (lane & 31));
                const uint32_t mine = keep16(p, drow, kbase, half);
                const int kl = lane & 31, reg = 4 * (kl >> 3) + (kl & 3), kh = (kl >> 2) & 1;
                uint32_t word = 0;
#pragma unroll
                for (int r = 0; r < 16; ++r) {
                    const unsigned long long bal = __ballot((mine >> r) & 1u);
                    const uint32_t part = kh ? (uint32_t)(bal >> 32) : (uint32_t)bal;
                    word = reg == r ? part : word;
                }
                keep = word;                                                  // bit: query of this 32-row block
            }
            f32x16 g = zero16();
#pragma unroll
            for (int s = 0; s < W / 16; ++s) g = mfma32(row_frag<W>(Os, qt * 32 + (lane & 31), 2 * s + half), vf[s], g);
            f32x16 a;
            f32x16 ds[2];
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                f32x16 s = zero16();
#pragma unroll
                for (int ks = 0; ks < NS; ++ks)
                    s = mfma32(row_frag<W>(Qs, qt * 32 + (lane & 31), (j * D + ks * 16) / 8 + half), kf[j][ks], s);
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const int at = qt * 32 + 8 * i + 4 * half;
                    const f32x4 m4 = *reinterpret_cast<const f32x4*>(&st[2 * j][at]);
                    const f32x4 l4 = *reinterpret_cast<const f32x4*>(&st[2 * j + 1][at]);
                    const f32x4 D4 = *reinterpret_cast<const f32x4*>(&st[4 + j][at]);
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const int r = 4 * i + e;
                        const float pr = __builtin_amdgcn_exp2f((__builtin_fmaf(s[r], p.sc, mk) - m4[e]) - l4[e]);
                        float gr = g[r];
                        if constexpr (DROP) gr = (keep >> (acc_row(r) + 4 * half)) & 1u ? gr * dscale : 0.f;
                        ds[j][r] = pr * (gr - D4[e]);
                        a[r] = j == 0 ? pr : a[r] - lam * pr;
                    }
                }
            }
            if constexpr (DROP) {
#pragma unroll
                for (int r = 0; r < 16; ++r) a[r] = (keep >> (acc_row(r) + 4 * half)) & 1u ? a[r] * dscale : 0.f;
            }
#pragma unroll
            for (int kk = 0; kk < 2; ++kk) {
                const bf16x8 af = pack_step(a, kk);
#pragma unroll
                for (int t = 0; t < NV; ++t) dv[t] = mfma32(tr_frag<W>(Os, qt * 32 + kk * 16, t * 32, lane), af, dv[t]);
#pragma unroll
                for (int j = 0; j < 2; ++j) {
                    const bf16x8 df = pack_step(ds[j], kk);
#pragma unroll
                    for (int t = 0; t < ND; ++t) dk[j][t] = mfma32(tr_frag<W>(Qs, qt * 32 + kk * 16, j * D + t * 32, lane), df, dk[j][t]);
                }
            }
        }
    }
    const float z = p.sc * (1.f / LOG2E);
    bf16_t* dkp = p.dk + (int64_t)b * p.bdk * (p.cu_k == nullptr) + (sk.row + key) * p.ldk + h * W;
    bf16_t* dvp = p.dv + (int64_t)b * p.bdv * (p.cu_k == nullptr) + (sk.row + key) * p.ldv + h * W;
#pragma unroll
    for (int t = 0; t < NV; ++t) store_block32(dvp + t * 32, dv[t], half, live);
#pragma unroll
    for (int j = 0; j < 2; ++j)
#pragma unroll
        for (int t = 0; t < ND; ++t) {
            dk[j][t] *= j == 0 ? z : -lam * z;
            store_block32(dkp + j * D + t * 32, dk[j][t], half, live);
        }
}

// ------------------------------------------------------------------------------------------------
// host side
// ------------------------------------------------------------------------------------------------
bool aligned16(const void* a) { return ((uintptr_t)a & 15) == 0; }

int check(const UniterDiffAttention* a) {
    UH_CHECK_ARG(a != nullptr, "null pointer");
    UH_CHECK_ARG(a->head_dim == 32 || a->head_dim == 64, "head_dim (width of one map's queries and keys) must be 32 or 64");
    UH_CHECK_ARG(a->B >= 0 && a->B <= (1 << 24) && a->heads >= 1 && a->heads <= 4096, "bad batch or head count");
    UH_CHECK_ARG(a->Lq >= 0 && a->Lk >= 0 && a->Lq <= (1 << 30) && a->Lk <= (1 << 30), "bad sequence length");
    UH_CHECK_ARG((a->cu_seqlens_q == nullptr) == (a->cu_seqlens_k == nullptr), "packed rows need cu_seqlens of both the queries and the keys");
    UH_CHECK_ARG(a->cu_seqlens_q == nullptr || a->mask_bias == nullptr, "packed rows take no mask");
    UH_CHECK_ARG(a->total_q >= 0 && a->total_k >= 0, "bad row count");
    UH_CHECK_ARG(a->p_drop >= 0.f && a->p_drop < 1.f, "dropout probability must be in [0,1)");
    UH_CHECK_ARG(a->q_row % 8 == 0 && a->k_row % 8 == 0 && a->v_row % 8 == 0 && a->q_batch % 8 == 0 && a->k_batch % 8 == 0 && a->v_batch % 8 == 0,
                 "row and batch strides must be multiples of 8 elements");
    UH_CHECK_ARG(aligned16(a->q) && aligned16(a->k) && aligned16(a->v) && aligned16(a->norm_weight), "q, k, v and norm_weight must be 16-byte aligned");
    UH_CHECK_ARG(a->lambda_q1 && a->lambda_k1 && a->lambda_q2 && a->lambda_k2, "null pointer");
    const int64_t blocks = a->B * a->heads * ((a->Lq > a->Lk ? a->Lq : a->Lk) / 32 + 1);
    UH_CHECK_ARG(blocks < ((int64_t)1 << 31), "too many tokens for one launch");
    return 0;
}

DiffArgs args_of(const UniterDiffAttention* a) {
    DiffArgs p{};
    p.q = (const bf16_t*)a->q; p.k = (const bf16_t*)a->k; p.v = (const bf16_t*)a->v;
    p.lq = a->q_row; p.lk = a->k_row; p.lv = a->v_row;
    p.bq = a->q_batch; p.bk = a->k_batch; p.bv = a->v_batch;
    p.mask = a->mask_bias; p.lmask = a->mask_row;
    p.cu_q = a->cu_seqlens_q; p.cu_k = a->cu_seqlens_k; p.tot_q = a->total_q; p.tot_k = a->total_k;
    p.lq1 = (const bf16_t*)a->lambda_q1; p.lk1 = (const bf16_t*)a->lambda_k1;
    p.lq2 = (const bf16_t*)a->lambda_q2; p.lk2 = (const bf16_t*)a->lambda_k2;
    p.lam_stride = a->lambda_per_head ? (int)a->head_dim : 0;
    p.lambda_init = a->lambda_init;
    p.w = (const bf16_t*)a->norm_weight; p.eps = a->norm_eps;
    p.B = (int)a->B; p.heads = (int)a->heads; p.Lq = (int)a->Lq; p.Lk = (int)a->Lk;
    p.sc = LOG2E / sqrtf((float)a->head_dim);
    p.drop = make_dropout(a->p_drop, a->seed, a->offset);
    return p;
}

// waves per workgroup: 32 rows each, up to four
int waves_for(int64_t L) { return (int)(L >= 97 ? 4 : (L + 31) / 32); }

int rows_per_chunk(const UniterDiffAttention* a) {
    // about 1024 workgroups over (head, chunk of rows); a chunk is whole passes of 32 rows
    const int64_t rows = a->B * a->Lq;
    int64_t per = (rows * a->heads + 1023) / 1024;
    per = (per + 31) / 32 * 32;
    return (int)(per < 32 ? 32 : per);
}

struct BwdSpace { size_t dctx, D, lam, w, bytes; int chunks, rows_per; };
BwdSpace bwd_space(const UniterDiffAttention* a) {
    BwdSpace s{};
    const int64_t rows = a->cu_seqlens_q != nullptr ? a->total_q : a->B * a->Lq;
    const int64_t W = 2 * a->head_dim;
    s.rows_per = rows_per_chunk(a);
    s.chunks = (int)((a->B * a->Lq + s.rows_per - 1) / s.rows_per);
    auto take = [&](size_t n) { const size_t at = s.bytes; s.bytes += (n + 255) & ~(size_t)255; return at; };
    s.dctx = take(a->norm_weight != nullptr ? (size_t)(rows * a->heads * W * 2) : 0);
    s.D = take((size_t)(a->B * a->heads * a->Lq * 2 * 4));
    s.lam = take((size_t)(a->heads * s.chunks * 4));
    s.w = take((size_t)(a->heads * s.chunks * W * 4));
    return s;
}

template <int D>
int launch_fwd(const DiffArgs& p, hipStream_t st) {
    const int nw = waves_for(p.Lq), nqb = (p.Lq + 32 * nw - 1) / (32 * nw);
    const dim3 grid((unsigned)(p.B * p.heads * nqb)), block(64 * nw);
    if (p.drop.p > 0.f) hipLaunchKernelGGL((diff_fwd_kernel<D, true>), grid, block, 0, st, p, nqb);
    else hipLaunchKernelGGL((diff_fwd_kernel<D, false>), grid, block, 0, st, p, nqb);
    UH_LAUNCH_CHECK();
    return 0;
}

template <int D>
int launch_bwd(const DiffArgs& p, const BwdSpace& s, const ParamGrads& g, hipStream_t st) {
    constexpr int W = 2 * D;
    if (s.chunks > 0) {
        hipLaunchKernelGGL((diff_bwd_rows_kernel<W>), dim3((unsigned)s.chunks, (unsigned)p.heads), dim3(256), 0, st, p, s.rows_per);
        UH_LAUNCH_CHECK();
    }
    const int nwq = waves_for(p.Lq), nqb = p.Lq > 0 ? (p.Lq + 32 * nwq - 1) / (32 * nwq) : 0;
    if (nqb > 0 && p.B > 0) {
        const dim3 grid((unsigned)(p.B * p.heads * nqb)), block(64 * nwq);
        if (p.drop.p > 0.f) hipLaunchKernelGGL((diff_bwd_dq_kernel<D, true>), grid, block, 0, st, p, nqb);
        else hipLaunchKernelGGL((diff_bwd_dq_kernel<D, false>), grid, block, 0, st, p, nqb);
        UH_LAUNCH_CHECK();
    }
    const int nwk = waves_for(p.Lk), nkb = p.Lk > 0 ? (p.Lk + 32 * nwk - 1) / (32 * nwk) : 0;
    if (nkb > 0 && p.B > 0) {
        const dim3 grid((unsigned)(p.B * p.heads * nkb)), block(64 * nwk);
        if (p.drop.p > 0.f) hipLaunchKernelGGL((diff_bwd_dkv_kernel<D, true>), grid, block, 0, st, p, nkb);
        else hipLaunchKernelGGL((diff_bwd_dkv_kernel<D, false>), grid, block, 0, st, p, nkb);
        UH_LAUNCH_CHECK();
    }
    const unsigned blocks = (unsigned)(g.n_lam + (g.w != nullptr ? W / 8 : 0));
    hipLaunchKernelGGL((diff_bwd_params_kernel<D>), dim3(blocks), dim3(256), 0, st, p, g);
    UH_LAUNCH_CHECK();
    return 0;
}

}  // namespace

extern "C" {

int uniter_diff_attention_fwd(const UniterDiffAttention* a, void* out, int64_t out_row, int64_t out_batch, float* stats, float* maps,
                              void* stream) {
    if (const int rc = check(a)) return rc;
    if (a->B == 0 || a->Lq == 0) return 0;
    UH_CHECK_ARG(a->q && out && (a->Lk == 0 || (a->k && a->v)), "null pointer");
    UH_CHECK_ARG(aligned16(out) && aligned16(stats) && aligned16(maps), "out, stats and maps must be 16-byte aligned");
    UH_CHECK_ARG(out_row % 8 == 0 && out_batch % 8 == 0, "row and batch strides must be multiples of 8 elements");
    UH_CHECK_ARG((stats == nullptr) == (maps == nullptr), "stats and maps are kept together, or neither");
    DiffArgs p = args_of(a);
    p.out = (bf16_t*)out; p.lo = out_row; p.bo = out_batch;
    p.stats = stats; p.maps = maps;
    return a->head_dim == 32 ? launch_fwd<32>(p, (hipStream_t)stream) : launch_fwd<64>(p, (hipStream_t)stream);
}

size_t uniter_diff_attention_bwd_workspace_bytes(const UniterDiffAttention* a) { return check(a) ? 0 : bwd_space(a).bytes; }

int uniter_diff_attention_bwd(const UniterDiffAttention* a, const float* stats, const float* maps, const void* dout, int64_t dout_row,
                              int64_t dout_batch, const UniterDiffAttentionGrads* g, void* workspace, size_t workspace_bytes, void* stream) {
    if (const int rc = check(a)) return rc;
    UH_CHECK_ARG(g != nullptr, "null pointer");
    UH_CHECK_ARG((a->norm_weight != nullptr) || g->norm_weight == nullptr, "a gradient of norm_weight needs norm_weight");
    const bool any = a->B > 0 && a->Lq > 0;
    UH_CHECK_ARG(!any || (a->q && stats && maps && dout && g->q && (a->Lk == 0 || (a->k && a->v))), "null pointer");
    UH_CHECK_ARG(a->B == 0 || a->Lk == 0 || (g->k && g->v), "null pointer");
    UH_CHECK_ARG(aligned16(stats) && aligned16(maps) && aligned16(dout) && aligned16(g->q) && aligned16(g->k) && aligned16(g->v) && aligned16(workspace),
                 "tensors must be 16-byte aligned");
    UH_CHECK_ARG((dout_row | dout_batch | g->q_row | g->k_row | g->v_row | g->q_batch | g->k_batch | g->v_batch) % 8 == 0,
                 "row and batch strides must be multiples of 8 elements");
    const BwdSpace s = bwd_space(a);
    UH_CHECK_ARG(workspace_bytes >= s.bytes && (workspace != nullptr || s.bytes == 0), "workspace too small");
    DiffArgs p = args_of(a);
    p.stats = const_cast<float*>(stats); p.maps = const_cast<float*>(maps);
    p.dout = (const bf16_t*)dout; p.ldo = dout_row; p.bdo = dout_batch;
    char* ws = (char*)workspace;
    p.dctx = a->norm_weight != nullptr ? (bf16_t*)(ws + s.dctx) : nullptr;
    p.D = (float*)(ws + s.D);
    p.part_lam = (float*)(ws + s.lam);
    p.part_w = (float*)(ws + s.w);
    p.chunks = s.chunks;
    p.dq = (bf16_t*)g->q; p.dk = (bf16_t*)g->k; p.dv = (bf16_t*)g->v;
    p.ldq = g->q_row; p.ldk = g->k_row; p.ldv = g->v_row;
    p.bdq = g->q_batch; p.bdk = g->k_batch; p.bdv = g->v_batch;
    ParamGrads pg;
    pg.lq1 = (bf16_t*)g->lambda_q1; pg.lk1 = (bf16_t*)g->lambda_k1; pg.lq2 = (bf16_t*)g->lambda_q2; pg.lk2 = (bf16_t*)g->lambda_k2;
    pg.w = (bf16_t*)g->norm_weight;
    pg.n_lam = a->lambda_per_head ? p.heads : 1;
    pg.accumulate = g->accumulate_params;
    return a->head_dim == 32 ? launch_bwd<32>(p, s, pg, (hipStream_t)stream) : launch_bwd<64>(p, s, pg, (hipStream_t)stream);
}

}  // extern "C"
