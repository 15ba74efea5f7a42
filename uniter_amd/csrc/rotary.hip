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
// What bounds it: HBM (4 bytes per element, ~1 flop).  One wave takes one token.  No table is read: a wave forms each pair's sine and
// cosine once (half a dozen 64-bit instructions per pair) and hands them round through LDS.  Measured: 32749 tokens of 24 heads of 64, half
// of each turned, 38.8 us (5.2 TB/s; 31 on inputs that the Infinity Cache partly holds, where a plain copy takes 28); with a lane holding
// both halves of 8 pairs (32-byte pieces of a row per load, each angle formed by every head's lanes) it was 52.7 us.  2848 tokens of 32
// heads: 6 us, of which 3.5 are the launch.  One token: 2.7 us in the kernel.
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
    const int64_t row = (int64_t)blockIdx.x * (blockDim.x >> 6) + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    if (row >= p.rows) return false;
    const int64_t b = p.rows >> 32 ? row / p.L : (uint32_t)row / p.L, l = row - b * p.L;      // (the 64-bit division is ten times as long)
    xo = b * p.xb + l * p.xl;
    yo = b * p.yb + l * p.yl;
    pos = (double)(p.pos != nullptr ? p.pos[b * p.pos_b + l] + p.pos_offset : l + p.pos_offset);
    return true;
}

// 16-byte accesses: every head starts on 16 bytes and the turned part is whole chunks of 8 pairs.  A lane takes one chunk of 8 elements of
// a head, 64 / (dim / 8) heads side by side, so that loads and stores run over whole rows.  The half layout's partners sit in the lane
// rot / 16 further on and come over a lane shuffle.
template <bool INTER>
__global__ __launch_bounds__(256) void rotary_kernel(const RotArgs p) {
    constexpr int N = 4;                                // heads in flight per lane
    int64_t xo, yo;
    double pos;
    if (!rot_row(p, xo, yo, pos)) return;
    const int lane = threadIdx.x & 63;
    const bf16_t* x = p.x + xo;
    bf16_t* y = p.y + yo;
    const int nj = p.rot >> 4, nc = p.dim >> 3, hs = 64 / nc;      // chunks of the turned halves and of a head; heads per pass
    const int h0 = lane / nc, ch = lane - h0 * nc;
    const bool turned = ch < 2 * nj, mine = h0 < hs && (turned || p.copy);
    x += ch * 8;
    y += ch * 8;
    u32x4 in[N] = {};
#pragma unroll
    for (int i = 0; i < N; ++i)
        if (const int h = h0 + i * hs; mine && h < p.heads) in[i] = ldg16<false>(x + h * p.xh);
    // every pair's cosine and sine once per token, passed round through the wave's own piece of LDS (no other wave touches it)
    extern __shared__ __attribute__((aligned(16))) float rot_lds[];
    float* const cs = rot_lds + (threadIdx.x >> 6) * p.rot;
    const int np = p.rot >> 1;
    for (int i = lane; i < np; i += 64) rot_angle(p, pos, i, cs[i], cs[np + i]);
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
    constexpr int W = INTER ? 4 : 8;                    // pairs that this lane's chunk has a part in
    const int pair = turned ? (INTER ? 4 * ch : 8 * (ch < nj ? ch : ch - nj)) : 0;
    const float sgn = !INTER && ch < nj ? -1.f : 1.f;
    const int mate = lane + (ch < nj ? nj : -nj);
    float c[W], s[W];
#pragma unroll
    for (int e = 0; e < W; ++e) {
        c[e] = turned ? cs[pair + e] : 1.f;
        s[e] = turned ? cs[np + pair + e] * sgn : 0.f;
    }
    for (int base = 0; base < p.heads; base += N * hs) {           // (the same for every lane: all take part in the shuffles)
#pragma unroll
        for (int i = 0; i < N; ++i) {
            if (base + i * hs >= p.heads) break;
            const int h = base + h0 + i * hs;
            const bool live = mine && h < p.heads;
            const u32x4 v = in[i];
            if (const int n = h + N * hs; mine && n < p.heads) in[i] = ldg16<false>(x + n * p.xh);
            float u[8], f[8];
            unpack8(v, u);
            if constexpr (INTER) {
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    f[2 * e] = u[2 * e] * c[e] - u[2 * e + 1] * s[e];
                    f[2 * e + 1] = u[2 * e + 1] * c[e] + u[2 * e] * s[e];
                }
            } else {
                u32x4 o;
#pragma unroll
                for (int e = 0; e < 4; ++e) o[e] = __builtin_amdgcn_ds_bpermute(mate << 2, v[e]);
                float w[8];
                unpack8(o, w);
#pragma unroll
                for (int e = 0; e < 8; ++e) f[e] = u[e] * c[e] + w[e] * s[e];
            }
            // plain stores: 2 microseconds of 53 faster than non-temporal ones for 32749 tokens of 24 heads
            if (live) *(gmem_u32x4*)(y + h * p.yh) = turned ? pack8(f) : v;
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

// ---- which elements a call touches: {b * s0 + l * s1 + h * s2 + [0, dim)}, dimensions of more than one with positive strides
struct Heads {
    int64_t at;                          // of the lowest element, in elements
    int64_t n[3], s[3];                  // by descending stride
    int dims;
    __int128 span[4];                    // from the lowest to the highest element of dimensions i .. dims - 1 and a head
    bool apart;                          // no two heads have an element in common (each stride is at least the span inside it)
};
Heads heads_of(const UniterRotary* r, const void* base, const int64_t* strides) {
    const int64_t sizes[3] = {r->B, r->L, r->heads};
    Heads a{};
    a.at = (int64_t)((uintptr_t)base >> 1);
    for (int i = 0; i < 3; ++i) {
        if (sizes[i] < 2) continue;
        int64_t s = strides[i];
        if (s < 0) { a.at += (sizes[i] - 1) * s; s = -s; }
        int at = a.dims++;
        for (; at > 0 && a.s[at - 1] < s; --at) { a.s[at] = a.s[at - 1]; a.n[at] = a.n[at - 1]; }
        a.s[at] = s;
        a.n[at] = sizes[i];
    }
    a.span[a.dims] = r->head_dim;
    a.apart = true;
    for (int i = a.dims - 1; i >= 0; --i) {
        a.apart = a.apart && a.s[i] >= a.span[i + 1];
        a.span[i] = (__int128)(a.n[i] - 1) * a.s[i] + a.span[i + 1];
    }
    return a;
}
// Whether heads of two such sets `delta` elements apart meet, both with a's sizes and strides (a.apart): some t with |t_i| < n_i has
// |delta + sum t_i s_i| < dim.  What the inner dimensions can still add is less than span[i + 1] <= s_i, so only the two t_i next to
// -delta / s_i come into question.
bool meet(const Heads& a, int i, __int128 delta) {
    if (i == a.dims) return delta < a.span[i] && -delta < a.span[i];
    __int128 t = -delta / a.s[i];
    if (t * a.s[i] > -delta) --t;                              // (rounded down)
    for (int k = 0; k < 2; ++k, ++t)
        if (t > -a.n[i] && t < a.n[i] && meet(a, i + 1, delta + t * a.s[i])) return true;
    return false;
}
// y is another tensor than x and they share an element.  Layouts that differ are taken to share one where their ranges meet.
bool overlap(const Heads& x, const Heads& y) {
    const __int128 delta = (__int128)y.at - x.at;
    if (delta >= x.span[0] || -delta >= y.span[0]) return false;
    bool alike = x.apart && x.dims == y.dims;
    for (int i = 0; alike && i < x.dims; ++i) alike = x.s[i] == y.s[i] && x.n[i] == y.n[i];
    return !alike || meet(x, 0, delta);
}

}  // namespace

extern "C" int uniter_rotary(const UniterRotary* r, const void* x, const int64_t* x_strides, void* y, const int64_t* y_strides,
                             void* stream) {
    UH_CHECK_ARG(r && x_strides && y_strides, "null pointer");
    UH_CHECK_ARG(r->B >= 0 && r->L >= 0 && r->L < ((int64_t)1 << 32) && r->heads >= 1 && r->heads <= 65536, "bad sizes");
    UH_CHECK_ARG(r->head_dim >= 2 && r->head_dim <= 1024, "head_dim must be 2 .. 1024");
    UH_CHECK_ARG(r->rot_dim >= 2 && r->rot_dim % 2 == 0 && r->rot_dim <= r->head_dim, "rot_dim must be even and at most head_dim");
    if (r->B == 0 || r->L == 0) return 0;
    UH_CHECK_ARG(x && y, "null pointer");
    const bool same = x == y && x_strides[0] == y_strides[0] && x_strides[1] == y_strides[1] && x_strides[2] == y_strides[2];
    UH_CHECK_ARG(same || x != y, "in place needs y's strides to be x's");
    // (a wave writes a token's heads while another may still read: any element in common would be a race)
    const Heads hy = heads_of(r, y, y_strides);
    UH_CHECK_ARG(hy.apart, "the heads of y overlap each other");
    UH_CHECK_ARG(same || !overlap(heads_of(r, x, x_strides), hy), "y overlaps x without being x");
    UH_CHECK_ARG(r->freq, "null pointer");
    UH_CHECK_ARG(((uintptr_t)r->freq & 7) == 0 && ((uintptr_t)r->positions & 7) == 0 && (((uintptr_t)x | (uintptr_t)y) & 1) == 0, "misaligned pointer");
    UH_CHECK_ARG(r->B <= ((int64_t)1 << 40) / r->L, "too many tokens");
    const int64_t rows = r->B * r->L;
    const int64_t blocks = (rows + 3) / 4;
    UH_CHECK_ARG(blocks < ((int64_t)1 << 24), "too many tokens for one launch");           // (a launch has fewer than 2^32 threads)
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
    p.copy = !same && p.dim > p.rot;
    const int64_t all = p.xb | p.xl | p.xh | p.yb | p.yl | p.yh | (p.copy ? p.dim : 0);
    const bool wide = p.dim % 8 == 0 && p.dim <= 512 && p.rot % 16 == 0 && all % 8 == 0 && (((uintptr_t)x | (uintptr_t)y) & 15) == 0;
    const hipStream_t st = (hipStream_t)stream;
    const dim3 grid((unsigned)blocks), block(rows < 4 ? 64 * (unsigned)rows : 256);
    const unsigned lds = (block.x >> 6) * (unsigned)p.rot * sizeof(float);      // at most 4 * 512 * 4 bytes
    if (wide) {
        if (r->interleaved) hipLaunchKernelGGL(rotary_kernel<true>, grid, block, lds, st, p);
        else hipLaunchKernelGGL(rotary_kernel<false>, grid, block, lds, st, p);
    } else {
        if (r->interleaved) hipLaunchKernelGGL(rotary_any_kernel<true>, grid, block, 0, st, p);
        else hipLaunchKernelGGL(rotary_any_kernel<false>, grid, block, 0, st, p);
    }
    UH_LAUNCH_CHECK();
    return 0;
}
