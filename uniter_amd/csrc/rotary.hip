// rotary.hip — rotary positions: the pairs of a head's first `rot_dim` elements turned by angles proportional to the token position.
//
//   y[a] = m (x[a] cos t - x[b] sin t),  y[b] = m (x[b] cos t + x[a] sin t),  t = position * freq[pair]
//   (a, b) = (i, rot_dim / 2 + i) in the half layout, (2 i, 2 i + 1) interleaved; elements from rot_dim on are copied.
//   The gradient of x is the same with -t: one kernel serves both directions (UniterRotary.inverse).
//
// Angles: freq holds TURNS per position (angle / 2 pi) in 64 bits.  position * freq is formed and reduced to its fraction in 64 bits —
// in 32 bits position 131071 would already be off by 0.008 of a radian — with the product's own rounding error added back, so that no
// position up to 2^53 loses anything; only the fraction goes to the 32-bit hardware sine and cosine, whose unit is the turn.
//
// What bounds it: HBM (4 bytes per element, ~1 flop).  One wave takes one token: lane = (head, chunk of 8 pairs), so a wave's loads
// cover whole rows, and a lane's eight sines and cosines are formed once and serve every head it comes to (nj = chunks per head divides
// the lanes into 64 / nj heads at a time).  No table is read: 8 angles per lane and token are ~60 vector instructions against the 128 to
// 512 bytes that the lane moves.
#include "common.cuh"
#include "kernels.h"
#include "../../include/uniter_hip.h"

namespace {

struct RotArgs {
    const bf16_t* x;
    bf16_t* y;
    int64_t xb, xl, xh, yb, yl, yh;      // strides in elements: batch, token, head
    const double* freq;
    const int64_t* pos;
    int64_t pos_b, pos_offset;
    int64_t rows;                        // B * L
    uint32_t L;
    int heads, dim, rot, copy;           // copy: elements from rot on are written too (y is not x)
    float mult, sign;
};

__device__ __forceinline__ void rot_angle(const RotArgs& p, const double pos, const int pair, float& c, float& s) {
    const double f = p.freq[pair], turns = pos * f;
    const float t = (float)(__builtin_amdgcn_fract(turns) + __builtin_fma(pos, f, -turns));      // (the second term: what the product lost)
    c = __builtin_amdgcn_cosf(t) * p.mult;
    s = __builtin_amdgcn_sinf(t) * p.mult * p.sign;
}

// the token of this wave; false behind the last one
__device__ __forceinline__ bool rot_row(const RotArgs& p, int64_t& xo, int64_t& yo, double& pos) {
    const int64_t row = (int64_t)blockIdx.x * (blockDim.x >> 6) + (threadIdx.x >> 6);
    if (row >= p.rows) return false;
    const int64_t b = row / p.L, l = row - b * p.L;
    xo = b * p.xb + l * p.xl;
    yo = b * p.yb + l * p.yl;
    pos = (double)(p.pos != nullptr ? p.pos[b * p.pos_b + l] + p.pos_offset : l + p.pos_offset);
    return true;
}

// 16-byte accesses: every head starts on 16 bytes and the turned part is whole chunks of 8 pairs
template <bool INTER>
__global__ __launch_bounds__(256) void rotary_kernel(const RotArgs p) {
    int64_t xo, yo;
    double pos;
    if (!rot_row(p, xo, yo, pos)) return;
    const int lane = threadIdx.x & 63;
    const bf16_t* x = p.x + xo;
    bf16_t* y = p.y + yo;
    const int nj = p.rot >> 4, hs = 64 / nj;            // chunks of 8 pairs per head; heads per pass
    const int j = lane % nj, h0 = lane / nj;
    const int oa = INTER ? 16 * j : 8 * j, ob = INTER ? 16 * j + 8 : p.rot / 2 + 8 * j;
    if (h0 < hs && h0 < p.heads) {
        u32x4 a = ldg16<false>(x + h0 * p.xh + oa), b = ldg16<false>(x + h0 * p.xh + ob);
        float c[8], s[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) rot_angle(p, pos, 8 * j + e, c[e], s[e]);
        for (int h = h0; h < p.heads; h += hs) {
            const u32x4 a0 = a, b0 = b;
            if (h + hs < p.heads) {                     // the next head's loads leave before this one's arithmetic
                a = ldg16<false>(x + (h + hs) * p.xh + oa);
                b = ldg16<false>(x + (h + hs) * p.xh + ob);
            }
            float u[8], v[8], fu[8], fv[8];
            unpack8(a0, u);
            unpack8(b0, v);
            if constexpr (INTER) {                      // pairs sit side by side: four in each piece
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    fu[2 * e] = u[2 * e] * c[e] - u[2 * e + 1] * s[e];
                    fu[2 * e + 1] = u[2 * e + 1] * c[e] + u[2 * e] * s[e];
                    fv[2 * e] = v[2 * e] * c[4 + e] - v[2 * e + 1] * s[4 + e];
                    fv[2 * e + 1] = v[2 * e + 1] * c[4 + e] + v[2 * e] * s[4 + e];
                }
            } else {
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    fu[e] = u[e] * c[e] - v[e] * s[e];
                    fv[e] = v[e] * c[e] + u[e] * s[e];
                }
            }
            out_store16(y + h * p.yh + oa, pack8(fu));
            out_store16(y + h * p.yh + ob, pack8(fv));
        }
    }
    if (p.copy) {
        const int nr = (p.dim - p.rot) >> 3;            // chunks of 8 elements per head that are not turned
        for (int e = lane; e < p.heads * nr; e += 64) {
            const int h = e / nr, c = e - h * nr;
            out_store16(y + h * p.yh + p.rot + c * 8, ldg16<false>(x + h * p.xh + p.rot + c * 8));
        }
    }
}

// any even rot_dim, any head size, any alignment: one pair per lane and step
template <bool INTER>
__global__ __launch_bounds__(256) void rotary_any_kernel(const RotArgs p) {
    int64_t xo, yo;
    double pos;
    if (!rot_row(p, xo, yo, pos)) return;
    const int lane = threadIdx.x & 63;
    const bf16_t* x = p.x + xo;
    bf16_t* y = p.y + yo;
    const int np = p.rot >> 1;
    for (int i = lane; i < np; i += 64) {
        float c, s;
        rot_angle(p, pos, i, c, s);
        const int oa = INTER ? 2 * i : i, ob = INTER ? 2 * i + 1 : np + i;
        for (int h = 0; h < p.heads; ++h) {
            const float u = bf2f(x[h * p.xh + oa]), v = bf2f(x[h * p.xh + ob]);
            y[h * p.yh + oa] = f2bf(u * c - v * s);
            y[h * p.yh + ob] = f2bf(v * c + u * s);
        }
    }
    if (p.copy) {
        const int nr = p.dim - p.rot;
        for (int e = lane; e < p.heads * nr; e += 64) {
            const int h = e / nr, c = e - h * nr;
            y[h * p.yh + p.rot + c] = x[h * p.xh + p.rot + c];
        }
    }
}

}  // namespace

extern "C" int uniter_rotary(const UniterRotary* r, const void* x, const int64_t* x_strides, void* y, const int64_t* y_strides,
                             void* stream) {
    UH_CHECK_ARG(r && x_strides && y_strides, "null pointer");
    UH_CHECK_ARG(r->B >= 0 && r->L >= 0 && r->L < ((int64_t)1 << 32) && r->heads >= 1 && r->heads <= 65536, "bad sizes");
    UH_CHECK_ARG(r->head_dim >= 2 && r->head_dim <= 1024, "head_dim must be 2 .. 1024");
    UH_CHECK_ARG(r->rot_dim >= 2 && r->rot_dim % 2 == 0 && r->rot_dim <= r->head_dim, "rot_dim must be even and at most head_dim");
    if (r->B == 0 || r->L == 0) return 0;
    UH_CHECK_ARG(x && y && r->freq, "null pointer");
    UH_CHECK_ARG(((uintptr_t)r->freq & 7) == 0 && ((uintptr_t)r->positions & 7) == 0 && (((uintptr_t)x | (uintptr_t)y) & 1) == 0, "misaligned pointer");
    UH_CHECK_ARG(r->B <= ((int64_t)1 << 40) / r->L, "too many tokens");
    const int64_t rows = r->B * r->L;
    const int64_t blocks = (rows + 3) / 4;
    UH_CHECK_ARG(blocks < ((int64_t)1 << 31), "too many tokens for one launch");
    RotArgs p;
    p.x = (const bf16_t*)x;
    p.y = (bf16_t*)y;
    p.xb = x_strides[0]; p.xl = x_strides[1]; p.xh = x_strides[2];
    p.yb = y_strides[0]; p.yl = y_strides[1]; p.yh = y_strides[2];
    p.freq = r->freq;
    p.pos = r->positions;
    p.pos_b = r->positions_batch_stride;
    p.pos_offset = r->position_offset;
    p.rows = rows;
    p.L = (uint32_t)r->L;
    p.heads = (int)r->heads; p.dim = (int)r->head_dim; p.rot = (int)r->rot_dim;
    p.mult = r->multiplier;
    p.sign = r->inverse ? -1.f : 1.f;
    const bool same = x == y && p.xb == p.yb && p.xl == p.yl && p.xh == p.yh;
    UH_CHECK_ARG(same || x != y, "in place needs y's strides to be x's");
    p.copy = !same && p.dim > p.rot;
    const int64_t all = p.xb | p.xl | p.xh | p.yb | p.yl | p.yh | (p.copy ? p.dim : 0);
    const bool wide = p.rot % 16 == 0 && all % 8 == 0 && (((uintptr_t)x | (uintptr_t)y) & 15) == 0;
    const hipStream_t st = (hipStream_t)stream;
    const dim3 grid((unsigned)blocks), block(rows < 4 ? 64 * (unsigned)rows : 256);
    if (wide) {
        if (r->interleaved) hipLaunchKernelGGL(rotary_kernel<true>, grid, block, 0, st, p);
        else hipLaunchKernelGGL(rotary_kernel<false>, grid, block, 0, st, p);
    } else {
        if (r->interleaved) hipLaunchKernelGGL(rotary_any_kernel<true>, grid, block, 0, st, p);
        else hipLaunchKernelGGL(rotary_any_kernel<false>, grid, block, 0, st, p);
    }
    UH_LAUNCH_CHECK();
    return 0;
}
