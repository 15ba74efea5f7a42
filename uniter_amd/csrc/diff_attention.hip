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
//
// Measured (MI355X; a library bf16 product of 8192^3 reaches 1200 TFLOP/s, a large copy 5.0 TB/s).  Forward, 12 d flops: 8192 keys d = 64
// 1000 TFLOP/s from 16 heads on, d = 32 870; 2048 keys 910 and 710 with 64 heads.  Backward, 28 d flops, 2048 keys and 64 heads: 670 (d = 32),
// 620 (d = 64).  The vector unit bounds it (two exponentials and about seven more instructions per query, key and map pair): forward at 8192
// keys it is busy 57 % of the SIMDs' cycles at d = 64 and the matrix cores 45 %, at d = 32 79 and 39 %: on one SIMD the two add up.  One
// query, 16381 keys, 4 x 12 heads: 36 us (5.5 TB/s) and 5 for the join.  32 x 96, 12 heads, d = 32: 10 us forward, 16 with what the backward
// pass wants kept, 8 + 23 backward: latency.  Dropout: two generator calls per lane and 32 keys, in all three loops (32 x 512, 12 heads,
// d = 32: forward 61 -> 100 us, backward 206 -> 252).
//
// Roundings to bf16, besides that of each result: the matrix cores take 16-bit operands, so what is formed in between and multiplied once more
// is rounded for them, each value once and by half a step (2^-9) at most — the weights exp(S - m) of the products with V (their sums l
// keep 32 bits), A = P_1 - lambda P_2 for dV, dS_1 / dS_2 for dQ and dK, and the norm's gradient dO for all three.  Products, maxima, sums,
// the maps' outputs kept for the backward pass, D and lambda are 32 bits.  Outputs are 2.5 - 2.7e-3 from the 64-bit result and gradients 3.0 -
// 3.3e-3, where 32 bits rounded once at the end give 1.7 - 1.9e-3.
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

// Division by a number that the host knows, for 0 <= n < 2^31: (n + high half of n mul) >> shift.  (The compiler's own takes 25
// instructions of code that every launch fetches cold.)
struct Div { uint32_t d, mul, shift; };
__device__ __forceinline__ int over(const int n, const Div v) { return (int)(((uint32_t)n + __umulhi((uint32_t)n, v.mul)) >> v.shift); }

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
    Div by_heads, by_Lq;
    float sc;                            // log2(e) / sqrt(d)
    DropoutCfg drop;
    bf16_t* out;                         // forward: rows [.., heads * W]
    int64_t lo, bo;
    float* stats;                        // [B, heads, Lq, NSTAT] or NULL
    float* maps;                         // [row, heads, 2, W]: P_1 V and P_2 V, or NULL
    float *psum, *pacc;                  // split forward: [split, B, heads, Lq, NSTAT] max and sum, [.., 2, W] sums not yet divided
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
// the larger one, or a NaN (one instruction for two of them: v_maximum3; fmaxf would quieten its operands first)
__device__ __forceinline__ float max2(const float a, const float b) { return __builtin_elementwise_maximum(a, b); }
// the value of lane ^ 32
__device__ __forceinline__ float other_half(const float x) {
    const uint32_t u = __float_as_uint(x);
    const auto s = __builtin_amdgcn_permlane32_swap(u, u, false, false);       // (lower half twice, upper half twice)
    return __uint_as_float((threadIdx.x & 32) ? s[0] : s[1]);
}
// row (or column) of an accumulator register: 8 (r / 4) + 4 half + r % 4
__device__ __forceinline__ constexpr int acc_row(const int r) { return 8 * (r >> 2) + (r & 3); }

// A lane holds columns 8 g + 4 half + {0..3}, g = 0..3, of one 32-column block of its row.  The two halves swap a group of every pair
// (v_permlane32_swap: the upper half of one register with the lower half of another), so that a lane stores 16 bytes: half 0 the 8 columns of the
// even group, half 1 those of the odd one.
__device__ __forceinline__ void store_block32(bf16_t* row, const f32x16& v, const int half, const bool valid) {
#pragma unroll
    for (int g = 0; g < 4; g += 2) {
        u32x4 w;
#pragma unroll
        for (int e = 0; e < 2; ++e) {
            const auto s = __builtin_amdgcn_permlane32_swap(pack_bf16x2(v[4 * g + 2 * e], v[4 * g + 2 * e + 1]),
                                                            pack_bf16x2(v[4 * g + 4 + 2 * e], v[4 * g + 4 + 2 * e + 1]), false, false);
            w[e] = s[0];
            w[2 + e] = s[1];
        }
        if (valid) out_store16(row + 8 * (g + half), w);
    }
}

// A kernel's arguments arrive through the scalar cache, cold, and the compiler asks for them where it needs them: five waits for memory one
// after the other before the first tile is under way.  One word of each of the N lines at once: the later loads hit.  (BYTES: of the
// arguments, which fill the lines up to there; the launch's own hidden ones follow.)
template <int BYTES>
__device__ __forceinline__ void warm_args() {
    typedef const __attribute__((address_space(4))) uint32_t* words;
    const words a = (words)__builtin_amdgcn_kernarg_segment_ptr();
    constexpr int N = (BYTES + 63) / 64;
    uint32_t x[N];
#pragma unroll
    for (int i = 0; i < N; ++i) x[i] = a[16 * i];
#pragma unroll
    for (int i = 0; i < N; ++i) asm volatile("" ::"s"(x[i]));
}

// Workgroups go to the 8 XCDs in turn.  `chunk` consecutive units of work (they share K and V, or Q and dO) stay on one XCD and its L2;
// successive chunks go to successive XCDs, so that sequences of different lengths spread over all of them.  The grid is padded to whole
// rounds of 8 chunks: an answer of `total` or more has nothing to do.
__device__ __forceinline__ int chunk_map(const int bid, const Div chunk) {
    const int loc = bid >> 3, c = over(loc, chunk), n = (int)chunk.d;
    return (c * 8 + (bid & 7)) * n + loc - c * n;
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

// additive mask in log2 units; the type's lowest value stays finite and above NONE, the reference of a row without keys yet (a row of
// nothing but lowest values is uniform over its keys)
constexpr float NONE = -3.4028234663852886e38f;
__device__ __forceinline__ float mask_log2(const float m) { return m == -INFINITY ? m : max2(m * LOG2E, -3e38f); }      // (a NaN stays one)

// ---- tiles by direct global -> LDS transfers (global_load_lds_dwordx4: a wave instruction moves 64 x 16 bytes to a contiguous 1 KiB
// of LDS, so the swizzle is applied to the source address).  The origin of a tile is scalar, a lane's offset inside it 32 bits (the entry
// checks the row strides).  Rows behind the end are read from the last row there is: their weight is zero, see zero_rows.
__device__ __forceinline__ uint32_t lds_addr(const void* p) {
    return (uint32_t)__builtin_amdgcn_readfirstlane((int)(uint32_t)(uintptr_t)(const __attribute__((address_space(3))) void*)p);
}
__device__ __forceinline__ void dma16(const uint32_t voff, const char* origin, const uint32_t lds) {
    asm volatile("s_mov_b32 m0, %2\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, %1" ::"v"(voff), "s"((__attribute__((address_space(1))) const char*)origin), "s"(lds) : "memory", "m0");
}
__device__ __forceinline__ void dma_wait() { asm volatile("s_waitcnt vmcnt(0)" ::: "memory"); }

// Values loaded before a loop are complete from here on: without it the compiler's wait for them (vmcnt, which counts the tile transfers
// too) lands inside the loop and waits for the next tile in every round.
template <int N>
__device__ __forceinline__ void pin(bf16x8 (&f)[N]) {
#pragma unroll
    for (int i = 0; i < N; ++i) asm volatile("" : "+v"(f[i]));
}

template <int W>
__device__ __forceinline__ void dma_tile(const bf16_t* tile, const bf16_t* src, const int64_t ld, const int r0, const int n, const int wid,
                                         const int nw, const int lane) {
    constexpr int RPI = 512 / W, CPR = W / 8;                  // rows per instruction, 16-byte chunks per row
    const char* origin = reinterpret_cast<const char*>(src + (int64_t)r0 * ld);
    const uint32_t base = lds_addr(tile), pitch = (uint32_t)(ld * 2);
    const int last = n - 1 - r0;
    for (int j = wid; j < KT / RPI; j += nw) {
        const int r = RPI * j + lane / CPR;
        const int key = W == 64 ? (((r >> 1) & 3) << 1) : ((r & 7) << 1);
        dma16((uint32_t)min(r, last) * pitch + (uint32_t)(((lane % CPR) ^ key) * 16), origin, base + (uint32_t)j * 1024u);
    }
}

// Masks of a tile's keys, one key per lane: prefetched with the tile, judged when it is there (the same in every wave).
struct TileMask {
    const float* row;                    // this example's row of the mask, or NULL
    int n;
    float m;                             // of the tile on its way
    bool general;                        // any key carries a mask
    unsigned long long out;              // keys that are out: -inf, or behind the end
    __device__ __forceinline__ void start(const int k0, const int lane) {
        if (row != nullptr) m = row[min(k0 + lane, n - 1)];
    }
    __device__ __forceinline__ float judge(const int k0, const int lane) {
        asm volatile("" : "+v"(m));      // (its own wait stays behind the transfers')
        const float mm = k0 + lane < n ? (row != nullptr ? mask_log2(m) : 0.f) : -INFINITY;
        general = __ballot(mm != 0.f) != 0;
        out = __ballot(mm == -INFINITY);
        return mm;
    }
};
// Rows that are out become zeros: whatever stands there, their weight is zero and 0 * NaN must not reach a sum.
template <int W>
__device__ __forceinline__ void zero_rows(bf16_t* tile, const unsigned long long out, const int tid, const int nthr) {
    for (int e = tid; e < KT * (W / 8); e += nthr) {
        const int r = e / (W / 8), c = e % (W / 8);
        if ((out >> r) & 1) *reinterpret_cast<u32x4*>(tile + tile_off<W>(r, c)) = u32x4{0u, 0u, 0u, 0u};
    }
}
// Key tiles up to the last one with a key that is not out (-inf): a padded batch's rear costs nothing.  All waves, the same answer.
__device__ __forceinline__ int live_tiles(const float* row, const int n, const int lane) {
    int nt = (n + KT - 1) / KT;
    if (row == nullptr || nt <= 2) return nt;
    while (nt > 0) {
        const int t0 = max(nt - 16, 0);
        float v[16];
#pragma unroll
        for (int i = 0; i < 16; ++i) v[i] = row[min((t0 + i) * KT + lane, n - 1)];
        int last = -1;
#pragma unroll
        for (int i = 0; i < 16; ++i)
            if (t0 + i < nt && __any(v[i] != -INFINITY)) last = i;             // (the last key, read again behind the end, is this tile's or later)
        if (last >= 0) return t0 + last + 1;
        nt = t0;
    }
    return 0;
}

// The key tiles of the forward and dQ kernels: K and V of KT keys, double buffered, and the keys' mask.
template <int W>
struct KeyTiles {
    bf16_t *Ks, *Vs;                     // [2][KT * W]
    float* mb;                           // [2][KT] additive mask, log2 units
    const bf16_t *K, *V;
    int64_t lk, lv;
    int wid, nw, lane;
    TileMask mk;

    __device__ __forceinline__ bf16_t* Kb(const int t) const { return Ks + (t & 1) * KT * W; }
    __device__ __forceinline__ bf16_t* Vb(const int t) const { return Vs + (t & 1) * KT * W; }
    __device__ __forceinline__ float* Mb(const int t) const { return mb + (t & 1) * KT; }
    __device__ __forceinline__ void start(const int t) {
        dma_tile<W>(Kb(t), K, lk, t * KT, mk.n, wid, nw, lane);
        dma_tile<W>(Vb(t), V, lv, t * KT, mk.n, wid, nw, lane);
        mk.start(t * KT, lane);
    }
    __device__ __forceinline__ void finish(const int t) {      // all waves: on return tile t is complete
        dma_wait();
        const float mm = mk.judge(t * KT, lane);
        if (mk.general && wid == 0) Mb(t)[lane] = mm;
        __syncthreads();
        if (mk.out != 0) {
            zero_rows<W>(Kb(t), mk.out, wid * 64 + lane, nw * 64);
            zero_rows<W>(Vb(t), mk.out, wid * 64 + lane, nw * 64);
            __syncthreads();
        }
    }
};

// a value that every lane has, in a scalar register
__device__ __forceinline__ float uniform(const float x) { return __uint_as_float((uint32_t)__builtin_amdgcn_readfirstlane((int)__float_as_uint(x))); }

// lambda of head h (every lane gets it)
template <int D>
__device__ __forceinline__ void lambda_of(const DiffArgs& p, const int h, const int lane, float& e1, float& e2) {
    float a = 0.f, b = 0.f;
    if (lane < D) {
        const int at = h * p.lam_stride + lane;
        a = bf2f(p.lq1[at]) * bf2f(p.lk1[at]);
        b = bf2f(p.lq2[at]) * bf2f(p.lk2[at]);
    }
    e1 = uniform(__expf(wave_sum(a)));
    e2 = uniform(__expf(wave_sum(b)));
}

// Random fields of the 16 elements (query of this lane, 32 keys from kb): word i holds those of registers 2 i and 2 i + 1; an element is kept
// when its field is at least drop.thresh.  One generator call covers the 8 registers of a 16-key step that one lane holds: group
// ((row * ceil(Lk / 16) + key / 16) * 2 + half).
struct Fields { uint32_t w[8]; };
__device__ __forceinline__ Fields fields16(const DiffArgs& p, const uint64_t row, const int kb, const int half) {
    const uint64_t n16 = (uint64_t)((p.Lk + 15) >> 4);
    const uint64_t g = (row * n16 + (uint64_t)(kb >> 4)) * 2 + (uint64_t)half;
    const u32x4 a = dropout_bits8(p.drop, g), b = dropout_bits8(p.drop, g + 2);
    Fields f;
#pragma unroll
    for (int i = 0; i < 4; ++i) { f.w[i] = a[i]; f.w[4 + i] = b[i]; }
    return f;
}
__device__ __forceinline__ bool kept(const DiffArgs& p, const Fields& f, const int r) {
    return (r & 1 ? f.w[r >> 1] >> 16 : f.w[r >> 1] & 0xffffu) >= p.drop.thresh;
}
// all ones in the halves of word i whose element is kept (packed 16-bit arithmetic: 0 from a saturated thresh - field, then 0 - 1)
__device__ __forceinline__ uint32_t keep_mask(const DiffArgs& p, const Fields& f, const int i) {
    typedef __attribute__((ext_vector_type(2))) unsigned short u16x2;
    const unsigned short t = (unsigned short)p.drop.thresh;
    const u16x2 x = __builtin_elementwise_sub_sat(u16x2{t, t}, __builtin_bit_cast(u16x2, f.w[i]));
    return __builtin_bit_cast(uint32_t, (u16x2)(__builtin_elementwise_min(x, u16x2{1, 1}) - u16x2{1, 1}));
}

// ------------------------------------------------------------------------------------------------
// forward
// ------------------------------------------------------------------------------------------------
// Rescaling of the accumulators waits until a score exceeds the reference maximum by 2^LAZY: until then the weights stay below 2^LAZY,
// whose bf16 operands are as exact as any others, and the reference need not be the maximum.
constexpr float LAZY = 8.f;

// A wave's 32 queries.  Blocks of 32 keys: scores S^T (both maps), weights, products with V.
template <int D>
struct FwdState {
    bf16x8 qf[2][D / 16];
    f32x16 o[2][D / 16];                 // [map][32 columns of V]
    float m[2], l[2];                    // reference (NONE: no key yet) and sum of the weights
    float se;                            // scores are s * se in log2 units (1 once a mask has been added)
};

template <int D>
__device__ __forceinline__ void fwd_scores(f32x16 (&s)[2], const FwdState<D>& f, const bf16_t* Kt, const int u, const int lane) {
    constexpr int W = 2 * D, NS = D / 16;
#pragma unroll
    for (int j = 0; j < 2; ++j) s[j] = zero16();
#pragma unroll
    for (int ks = 0; ks < NS; ++ks)
#pragma unroll
        for (int j = 0; j < 2; ++j)
            s[j] = mfma32(row_frag<W>(Kt, u * 32 + (lane & 31), (j * D + ks * 16) / 8 + (lane >> 5)), f.qf[j][ks], s[j]);
}
template <int D>
__device__ __forceinline__ void fwd_products(FwdState<D>& f, const bf16x8 (&pf)[2][2], const bf16_t* Vt, const int u, const int lane) {
    constexpr int W = 2 * D, NV = W / 32;
#pragma unroll
    for (int t = 0; t < NV; ++t)
#pragma unroll
        for (int kk = 0; kk < 2; ++kk) {
            const bf16x8 vf = tr_frag<W>(Vt, u * 32 + kk * 16, t * 32, lane);
            f.o[0][t] = mfma32(vf, pf[0][kk], f.o[0][t]);
            f.o[1][t] = mfma32(vf, pf[1][kk], f.o[1][t]);
        }
}
// The scores of a block have arrived: add the mask, and rows where one exceeds the reference maximum by 2^LAZY take a new one.
template <int D>
__device__ __forceinline__ void fwd_arrive(FwdState<D>& f, f32x16 (&s)[2], const DiffArgs& p, const float* mb, const bool general, const int u,
                                           const int lane) {
    const int half = lane >> 5;
    f.se = p.sc;
    if (general) {
        f.se = 1.f;
#pragma unroll
        for (int g = 0; g < 4; ++g) {
            const f32x4 mv = *reinterpret_cast<const f32x4*>(mb + u * 32 + 8 * g + 4 * half);
#pragma unroll
            for (int j = 0; j < 2; ++j)
#pragma unroll
                for (int e = 0; e < 4; ++e) s[j][4 * g + e] = __builtin_fmaf(s[j][4 * g + e], p.sc, mv[e]);
        }
    }
    float mx[2];
#pragma unroll
    for (int j = 0; j < 2; ++j) {
        mx[j] = max2(s[j][0], s[j][1]);
#pragma unroll
        for (int r = 2; r < 16; r += 2) mx[j] = max2(max2(mx[j], s[j][r]), s[j][r + 1]);
        mx[j] *= f.se;
    }
    if (__any(mx[0] > f.m[0] + LAZY || mx[1] > f.m[1] + LAZY)) {
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            const float top = max2(mx[j], other_half(mx[j]));
            const bool move = top > f.m[j] + LAZY;
            const float alpha = move ? __builtin_amdgcn_exp2f(f.m[j] - top) : 1.f;
            f.m[j] = move ? top : f.m[j];
            f.l[j] *= alpha;
#pragma unroll
            for (int t = 0; t < D / 16; ++t) f.o[j][t] *= alpha;
        }
    }
}
template <int D, bool DROP>
__device__ __forceinline__ void fwd_weights(FwdState<D>& f, f32x16 (&s)[2], bf16x8 (&pf)[2][2], const uint32_t (&keep)[8]) {
#pragma unroll
    for (int j = 0; j < 2; ++j) {
        float sum[2];
#pragma unroll
        for (int r = 0; r < 16; ++r) {
            s[j][r] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[j][r], f.se, -f.m[j]));
            sum[r & 1] = r < 2 ? s[j][r] : sum[r & 1] + s[j][r];
        }
        f.l[j] += sum[0] + sum[1];
#pragma unroll
        for (int kk = 0; kk < 2; ++kk) {
            pf[j][kk] = pack_step(s[j], kk);
            if constexpr (DROP) {
                u32x4 w = __builtin_bit_cast(u32x4, pf[j][kk]);
#pragma unroll
                for (int i = 0; i < 4; ++i) w[i] &= keep[4 * kk + i];
                pf[j][kk] = __builtin_bit_cast(bf16x8, w);
            }
        }
    }
}

struct FwdGrid { Div nqb, ns, chunk; int total; };             // query blocks per (example, head), splits, units per chunk; units

// one workgroup: `nw` waves of 32 queries each, key tiles [t0, t1) of its split.  SPLIT: writes partial sums for diff_join_kernel.
template <int D, bool DROP, bool SPLIT>
__global__ __launch_bounds__(256, D == 32 ? 3 : 2) void diff_fwd_kernel(const DiffArgs p, const FwdGrid g) {
    constexpr int W = 2 * D, NS = D / 16, NV = W / 32;
    __shared__ __attribute__((aligned(16))) bf16_t Ks[2 * KT * W];
    __shared__ __attribute__((aligned(16))) bf16_t Vs[2 * KT * W];
    __shared__ __attribute__((aligned(16))) float mb[2 * KT];
    warm_args<sizeof(DiffArgs) + sizeof(FwdGrid)>();
    const int bid = chunk_map((int)blockIdx.x, g.chunk);
    if (bid >= g.total) return;
    const int nsplit = (int)g.ns.d, unit = SPLIT ? over(bid, g.ns) : bid, sp = SPLIT ? bid - unit * nsplit : 0;
    const int bh = over(unit, g.nqb), qb = unit - bh * (int)g.nqb.d;
    const int b = over(bh, p.by_heads), h = bh - b * p.heads;
    const Span sq = span_of(p.cu_q, p.tot_q, b, p.Lq), sk = span_of(p.cu_k, p.tot_k, b, p.Lk);
    const int lane = threadIdx.x & 63, wid = __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6)), half = lane >> 5;
    const int nw = (int)blockDim.x >> 6, tid = (int)threadIdx.x;
    if (qb * nw * 32 >= sq.n) return;
    const int q = (qb * nw + wid) * 32 + (lane & 31);
    const bool live = q < sq.n, idle = q - (lane & 31) >= sq.n;                // (idle: a wave without rows helps with the tiles)
    KeyTiles<W> kt;
    kt.Ks = Ks; kt.Vs = Vs; kt.mb = mb;
    kt.K = p.k + (int64_t)b * p.bk * (p.cu_k == nullptr) + sk.row * p.lk + h * W;
    kt.V = p.v + (int64_t)b * p.bv * (p.cu_k == nullptr) + sk.row * p.lv + h * W;
    kt.lk = p.lk; kt.lv = p.lv;
    kt.wid = wid; kt.nw = nw; kt.lane = lane;
    kt.mk.row = p.mask != nullptr ? p.mask + (int64_t)b * p.lmask : nullptr;
    kt.mk.n = sk.n;
    kt.mk.m = 0.f;
    int t0 = 0, t1 = (sk.n + KT - 1) / KT;
    if constexpr (SPLIT) {
        t0 = (int)((int64_t)t1 * sp / nsplit);
        t1 = (int)((int64_t)t1 * (sp + 1) / nsplit);
    }
    if (t0 < t1) kt.start(t0);

    const bf16_t* Q = p.q + (int64_t)b * p.bq * (p.cu_q == nullptr) + (sq.row + min(q, sq.n - 1)) * p.lq + h * W + half * 8;
    FwdState<D> f;
#pragma unroll
    for (int j = 0; j < 2; ++j) {
#pragma unroll
        for (int s = 0; s < NS; ++s) f.qf[j][s] = __builtin_bit_cast(bf16x8, ldg16<false>(Q + j * D + s * 16));
        f.m[j] = NONE;
        f.l[j] = 0.f;
#pragma unroll
        for (int t = 0; t < NV; ++t) f.o[j][t] = zero16();
    }
    int touch = 0;
    if (!SPLIT && p.w != nullptr) touch = reinterpret_cast<const int*>(p.w)[lane & (D - 1)];      // (the epilogue's weights: into the cache)
    float e1, e2;
    lambda_of<D>(p, h, lane, e1, e2);
    if constexpr (!SPLIT) asm volatile("" ::"v"(touch));
    const float lam = e1 - e2 + p.lambda_init;
    const uint64_t drow = (uint64_t)bh * (uint64_t)p.Lq + (uint64_t)q;
    if (t0 < t1) t1 = min(t1, live_tiles(kt.mk.row, sk.n, lane));
    pin(f.qf[0]);
    pin(f.qf[1]);

    if (t0 < t1) kt.finish(t0);
    else dma_wait();                     // (a first tile whose keys are all out is on its way to LDS all the same)
    for (int t = t0; t < t1; ++t) {
        const bool general = kt.mk.general;
        const int subs = idle || kt.mk.out == ~0ull ? 0 : min(2, (sk.n - t * KT + 31) >> 5);
        if (t + 1 < t1) kt.start(t + 1);
        for (int u = 0; u < subs; ++u) {
            f32x16 s[2];
            bf16x8 pf[2][2];
            fwd_scores<D>(s, f, kt.Kb(t), u, lane);
            fwd_arrive<D>(f, s, p, kt.Mb(t), general, u, lane);
            uint32_t keep[8];
            if constexpr (DROP) {
                const Fields fl = fields16(p, drow, t * KT + u * 32, half);
#pragma unroll
                for (int i = 0; i < 8; ++i) keep[i] = keep_mask(p, fl, i);
            }
            fwd_weights<D, DROP>(f, s, pf, keep);
            fwd_products<D>(f, pf, kt.Vb(t), u, lane);
        }
        if (t + 1 < t1) kt.finish(t + 1);
    }
    f32x16(&o)[2][NV] = f.o;
    float(&m)[2] = f.m;
    float(&l)[2] = f.l;
#pragma unroll
    for (int j = 0; j < 2; ++j) {
        l[j] += other_half(l[j]);
        m[j] = m[j] == NONE ? 0.f : m[j];
    }
    const float dscale = DROP ? p.drop.scale : 1.f;
    if constexpr (SPLIT) {
        if (!live) return;
        const int64_t at = ((int64_t)sp * p.B * p.heads + bh) * p.Lq + q;
        if (half == 0) *reinterpret_cast<f32x4*>(p.psum + at * NSTAT) = f32x4{m[0], l[0], m[1], l[1]};
#pragma unroll
        for (int j = 0; j < 2; ++j)
#pragma unroll
            for (int t = 0; t < NV; ++t) {
                o[j][t] *= dscale;
                float* dst = p.pacc + (at * 2 + j) * W + t * 32 + 4 * half;
#pragma unroll
                for (int g = 0; g < 4; ++g) *reinterpret_cast<f32x4*>(dst + 8 * g) = f32x4{o[j][t][4 * g], o[j][t][4 * g + 1], o[j][t][4 * g + 2], o[j][t][4 * g + 3]};
            }
        return;
    }
    float inv[2];
#pragma unroll
    for (int j = 0; j < 2; ++j) inv[j] = l[j] > 0.f ? dscale / l[j] : l[j];    // (0 without keys; a NaN stays one)
    if (p.stats != nullptr && live && half == 0)
        *reinterpret_cast<f32x4*>(p.stats + ((int64_t)bh * p.Lq + q) * NSTAT) =
            f32x4{m[0], l[0] == 0.f ? INFINITY : __log2f(l[0]), m[1], l[1] == 0.f ? INFINITY : __log2f(l[1])};
    const int64_t row = p.cu_q != nullptr ? sq.row + q : (int64_t)b * p.Lq + q;
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
            for (int g = 0; g < 4; ++g) {
                float w4[4];
                unpack4(ldg8<false>(p.w + t * 32 + 8 * g + 4 * half), w4);
#pragma unroll
                for (int e = 0; e < 4; ++e) o[0][t][4 * g + e] *= rs * w4[e];
            }
    }
    bf16_t* out = p.out + (int64_t)b * p.bo * (p.cu_q == nullptr) + (sq.row + q) * p.lo + h * W;
#pragma unroll
    for (int t = 0; t < NV; ++t) store_block32(out + t * 32, o[0][t], half, live);
}

// lambda of head h from the W / 8 lanes of a row's group, four or so products each (every lane of the group gets it)
template <int D>
__device__ __forceinline__ float lambda_of_group(const DiffArgs& p, const int h, const int i) {
    constexpr int LN = 2 * D / 8, PER = D / LN;
    float a = 0.f, b = 0.f;
#pragma unroll
    for (int e = 0; e < PER; ++e) {
        const int at = h * p.lam_stride + i * PER + e;
        a += bf2f(p.lq1[at]) * bf2f(p.lk1[at]);
        b += bf2f(p.lq2[at]) * bf2f(p.lk2[at]);
    }
#pragma unroll
    for (int x = 1; x < LN; x <<= 1) { a += __shfl_xor(a, x, WAVE); b += __shfl_xor(b, x, WAVE); }
    return __expf(a) - __expf(b) + p.lambda_init;
}

// Joins the splits of a row (example, head, query): W / 8 lanes of 8 columns.  Few splits: every such group of lanes has a row of its own;
// many (GS > 1): GS groups share the splits of a row.  HBM bound: 102 MB in 19 us (8191 rows x 6 heads, d = 64, 2 splits).
template <int D, int GS>
__global__ __launch_bounds__(256) void diff_join_kernel(const DiffArgs p, const int nsplit) {
    constexpr int W = 2 * D, LN = W / 8;
    warm_args<sizeof(DiffArgs) + 4>();
    const int lane = threadIdx.x & 63, li = lane % LN, c = li * 8, gi = (lane / LN) % GS;
    const int64_t rows = (int64_t)p.B * p.heads * p.Lq;
    const int64_t r = ((int64_t)blockIdx.x * blockDim.x + threadIdx.x) / (LN * GS);
    const int64_t rc = r < rows ? r : rows - 1;                // (no lane leaves: the exchanges below are wave operations)
    const int bh = over((int)rc, p.by_Lq), q = (int)rc - bh * p.Lq, b = over(bh, p.by_heads), h = bh - b * p.heads;
    const Span sq = span_of(p.cu_q, p.tot_q, b, p.Lq);
    const bool live = r < rows && q < sq.n;
    float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f}, o[2][8];
#pragma unroll
    for (int j = 0; j < 2; ++j)
#pragma unroll
        for (int e = 0; e < 8; ++e) o[j][e] = 0.f;
    for (int s = live ? gi : nsplit; s < nsplit; s += GS) {    // (a row behind its example has no partial sums)
        const int64_t at = s * rows + rc;
        const f32x4 st = *reinterpret_cast<const f32x4*>(p.psum + at * NSTAT);
        f32x4 a[2][2];
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            a[j][0] = *reinterpret_cast<const f32x4*>(p.pacc + (at * 2 + j) * W + c);
            a[j][1] = *reinterpret_cast<const f32x4*>(p.pacc + (at * 2 + j) * W + c + 4);
        }
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            const float ls = st[2 * j + 1];
            const float mn = ls == 0.f ? m[j] : fmaxf(m[j], st[2 * j]);        // (a split without keys says nothing)
            const float f0 = m[j] == mn ? 1.f : __builtin_amdgcn_exp2f(m[j] - mn), f1 = ls == 0.f ? 0.f : __builtin_amdgcn_exp2f(st[2 * j] - mn);
            m[j] = mn;
            l[j] = l[j] * f0 + ls * f1;
#pragma unroll
            for (int e = 0; e < 8; ++e) o[j][e] = o[j][e] * f0 + a[j][e >> 2][e & 3] * f1;
        }
    }
    const float lam = lambda_of_group<D>(p, h, li);
#pragma unroll
    for (int x = LN; x < LN * GS; x <<= 1)
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            const float m2 = __shfl_xor(m[j], x, WAVE), l2 = __shfl_xor(l[j], x, WAVE), mn = fmaxf(m[j], m2);
            const float f0 = m[j] == mn ? 1.f : __builtin_amdgcn_exp2f(m[j] - mn), f1 = m2 == mn ? 1.f : __builtin_amdgcn_exp2f(m2 - mn);
            m[j] = mn;
            l[j] = l[j] * f0 + l2 * f1;
#pragma unroll
            for (int e = 0; e < 8; ++e) o[j][e] = o[j][e] * f0 + __shfl_xor(o[j][e], x, WAVE) * f1;
        }
    const int64_t row = p.cu_q != nullptr ? sq.row + q : (int64_t)b * p.Lq + q;
    const bool writes = live && gi == 0;
    float ss = 0.f;
#pragma unroll
    for (int j = 0; j < 2; ++j) {
        m[j] = m[j] == -INFINITY ? 0.f : m[j];
        const float inv = l[j] > 0.f ? 1.f / l[j] : l[j];
#pragma unroll
        for (int e = 0; e < 8; ++e) o[j][e] *= inv;
        if (p.maps != nullptr && writes) {
            float* at = p.maps + ((row * p.heads + h) * 2 + j) * W + c;
            *reinterpret_cast<f32x4*>(at) = f32x4{o[j][0], o[j][1], o[j][2], o[j][3]};
            *reinterpret_cast<f32x4*>(at + 4) = f32x4{o[j][4], o[j][5], o[j][6], o[j][7]};
        }
    }
    if (p.stats != nullptr && writes && li == 0)
        *reinterpret_cast<f32x4*>(p.stats + r * NSTAT) = f32x4{m[0], l[0] == 0.f ? INFINITY : __log2f(l[0]), m[1], l[1] == 0.f ? INFINITY : __log2f(l[1])};
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        o[0][e] -= lam * o[1][e];
        ss += o[0][e] * o[0][e];
    }
    if (p.w != nullptr) {
#pragma unroll
        for (int x = 1; x < LN; x <<= 1) ss += __shfl_xor(ss, x, WAVE);
        const float rs = rsqrtf(ss * (1.f / W) + p.eps) * (1.f - p.lambda_init);
        float w8[8];
        unpack8(ldg16<false>(p.w + c), w8);
#pragma unroll
        for (int e = 0; e < 8; ++e) o[0][e] *= rs * w8[e];
    }
    if (writes) out_store16(p.out + (int64_t)b * p.bo * (p.cu_q == nullptr) + (sq.row + q) * p.lo + h * W + c, pack8(o[0]));
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
    warm_args<sizeof(DiffArgs) + 4>();
    const int h = (int)blockIdx.y;
    const int c = ((int)threadIdx.x % LN) * 8, ri = (int)threadIdx.x / LN;
    const float lam = lambda_of_group<W / 2>(p, h, (int)threadIdx.x % LN), so = 1.f - p.lambda_init;
    float wv[8], aw[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f}, al = 0.f;
    if (p.w != nullptr) unpack8(*reinterpret_cast<const u32x4*>(p.w + c), wv);
    // rows are counted over all examples: (b, q), q < Lq
    const int64_t total = (int64_t)p.B * p.Lq;
    const int64_t r0 = (int64_t)blockIdx.x * rows_per;
    for (int i = ri; i < rows_per; i += RP) {
        const int64_t rr = r0 + i;
        const int b = over((int)rr, p.by_Lq), q = (int)rr - b * p.Lq;
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
        // The products that follow take dO as a bf16 operand, and D is formed from the same rounded values: what all v have in common cancels
        // in G - D only so (130 x 130, d = 32, v = noise + 16: dQ 3.0e-3 from the 64-bit result, with D from before the rounding 4.7e-2;
        // costs 0.1 - 0.2 us).  dlambda = -sum D_2 takes no difference and keeps the 32 bits.
        const u32x4 db = pack8(d);
        float dr[8], d1 = 0.f, d2 = 0.f;
        unpack8(db, dr);
#pragma unroll
        for (int e = 0; e < 8; ++e) { d1 += dr[e] * o1[e]; d2 += dr[e] * o2[e]; }
#pragma unroll
        for (int s = 1; s < LN; s <<= 1) { d1 += __shfl_xor(d1, s, WAVE); d2 += __shfl_xor(d2, s, WAVE); }
        if (ok) {
#pragma unroll
            for (int e = 0; e < 8; ++e) al -= d[e] * o2[e];
            if (p.dctx != nullptr) *reinterpret_cast<u32x4*>(p.dctx + (row * p.heads + h) * W + c) = db;
            if (c == 0) {
                float* D = p.D + (((int64_t)b * p.heads + h) * p.Lq + q) * 2;
                D[0] = d1;
                D[1] = d2;
            }
        }
    }
#pragma unroll
    for (int s = 1; s < LN; s <<= 1) al += __shfl_xor(al, s, WAVE);
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
__device__ __forceinline__ void bwd_params_block(const DiffArgs& p, const ParamGrads& g, const int bid, float* red) {
    constexpr int W = 2 * D;
    const int tid = (int)threadIdx.x, nthr = (int)blockDim.x, lane = tid & 63, wid = tid >> 6, nw = nthr >> 6;
    if (bid < g.n_lam) {
        const int64_t n = (int64_t)p.chunks * (g.n_lam == 1 ? p.heads : 1);
        const float* src = p.part_lam + (g.n_lam == 1 ? 0 : (int64_t)bid * p.chunks);
        float s = 0.f;
        for (int64_t i = tid; i < n; i += nthr) s += src[i];
        s = wave_sum(s);
        if (lane == 0) red[wid] = s;
        __syncthreads();
        if (tid < 64) {
            float e1, e2;
            lambda_of<D>(p, bid, tid, e1, e2);
            float sum = 0.f;
            for (int i = 0; i < nw; ++i) sum += red[i];
            const float d1 = sum * e1, d2 = -sum * e2;
            if (tid < D) {
                const int at = bid * p.lam_stride + tid;
                auto put = [&](bf16_t* dst, float v) { if (dst != nullptr) dst[at] = f2bf(g.accumulate ? bf2f(dst[at]) + v : v); };
                put(g.lq1, d1 * bf2f(p.lk1[at]));
                put(g.lk1, d1 * bf2f(p.lq1[at]));
                put(g.lq2, d2 * bf2f(p.lk2[at]));
                put(g.lk2, d2 * bf2f(p.lq2[at]));
            }
        }
        return;
    }
    const int c = (bid - g.n_lam) * 8 + (tid & 7);
    float s = 0.f;
    for (int64_t i = tid >> 3; i < (int64_t)p.heads * p.chunks; i += nthr >> 3) s += p.part_w[i * W + c];
#pragma unroll
    for (int x = 8; x < 64; x <<= 1) s += __shfl_xor(s, x, WAVE);
    if (lane < 8) red[wid * 8 + lane] = s;
    __syncthreads();
    if (tid < 8) {
        float sum = 0.f;
        for (int i = 0; i < nw; ++i) sum += red[i * 8 + tid];
        g.w[c] = f2bf(g.accumulate ? bf2f(g.w[c]) + sum : sum);
    }
}

// ------------------------------------------------------------------------------------------------
// backward, queries: dQ_j = sum_k dS_j K_j,  dS_1 = P_1 (G - D_1) / sqrt(d),  dS_2 = -lambda P_2 (G - D_2) / sqrt(d),  G = dropout(dO V^T)
// ------------------------------------------------------------------------------------------------
template <int D, bool DROP>
__device__ __forceinline__ void bwd_dq_block(const DiffArgs& p, const Div nqb, const int bid, char* smem) {
    constexpr int W = 2 * D, NS = D / 16, ND = D / 32;
    bf16_t *Ks = reinterpret_cast<bf16_t*>(smem), *Vs = Ks + 2 * KT * W;
    float* mb = reinterpret_cast<float*>(Vs + 2 * KT * W);
    const int bh = over(bid, nqb), qb = bid - bh * (int)nqb.d;
    const int b = over(bh, p.by_heads), h = bh - b * p.heads;
    const Span sq = span_of(p.cu_q, p.tot_q, b, p.Lq), sk = span_of(p.cu_k, p.tot_k, b, p.Lk);
    const int lane = threadIdx.x & 63, wid = __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6)), half = lane >> 5;
    const int nw = (int)blockDim.x >> 6;
    if (qb * nw * 32 >= sq.n) return;
    const int q = (qb * nw + wid) * 32 + (lane & 31);
    const bool live = q < sq.n, idle = q - (lane & 31) >= sq.n;
    const int qs = min(q, sq.n - 1);
    int nt = (sk.n + KT - 1) / KT;

    KeyTiles<W> kt;
    kt.Ks = Ks; kt.Vs = Vs; kt.mb = mb;
    kt.K = p.k + (int64_t)b * p.bk * (p.cu_k == nullptr) + sk.row * p.lk + h * W;
    kt.V = p.v + (int64_t)b * p.bv * (p.cu_k == nullptr) + sk.row * p.lv + h * W;
    kt.lk = p.lk; kt.lv = p.lv;
    kt.wid = wid; kt.nw = nw; kt.lane = lane;
    kt.mk.row = p.mask != nullptr ? p.mask + (int64_t)b * p.lmask : nullptr;
    kt.mk.n = sk.n;
    kt.mk.m = 0.f;
    if (nt > 0) kt.start(0);

    const bf16_t* Q = p.q + (int64_t)b * p.bq * (p.cu_q == nullptr) + (sq.row + qs) * p.lq + h * W + half * 8;
    const bf16_t* dO = p.dctx != nullptr ? p.dctx + (((p.cu_q != nullptr ? sq.row : (int64_t)b * p.Lq) + qs) * p.heads + h) * W
                                         : p.dout + (int64_t)b * p.bdo * (p.cu_q == nullptr) + (sq.row + qs) * p.ldo + h * W;
    bf16x8 qf[2][NS], gf[W / 16];
#pragma unroll
    for (int s = 0; s < W / 16; ++s) {
        qf[s / NS][s % NS] = __builtin_bit_cast(bf16x8, ldg16<false>(Q + s * 16));
        gf[s] = __builtin_bit_cast(bf16x8, ldg16<false>(dO + s * 16 + half * 8));
    }
    const f32x4 st = *reinterpret_cast<const f32x4*>(p.stats + ((int64_t)bh * p.Lq + qs) * NSTAT);
    const float m[2] = {st[0], st[2]}, ll[2] = {st[1], st[3]};
    // with dropout: G without its factor `dscale`, D over dscale, and dscale with the other factors at the end
    const float dscale = DROP ? p.drop.scale : 1.f, iscale = DROP ? 1.f / p.drop.scale : 1.f;
    float Dq[2] = {p.D[((int64_t)bh * p.Lq + qs) * 2] * iscale, p.D[((int64_t)bh * p.Lq + qs) * 2 + 1] * iscale};
    float e1, e2;
    lambda_of<D>(p, h, lane, e1, e2);
    const float lam = e1 - e2 + p.lambda_init;
    const uint64_t drow = (uint64_t)bh * (uint64_t)p.Lq + (uint64_t)q;

    f32x16 dq[2][ND];
#pragma unroll
    for (int j = 0; j < 2; ++j)
#pragma unroll
        for (int t = 0; t < ND; ++t) dq[j][t] = zero16();
    if (nt > 0) nt = live_tiles(kt.mk.row, sk.n, lane);
    pin(qf[0]);
    pin(qf[1]);
    pin(gf);
    float c_lse[2] = {m[0] + ll[0], m[1] + ll[1]};
    asm volatile("" : "+v"(c_lse[0]), "+v"(c_lse[1]), "+v"(Dq[0]), "+v"(Dq[1]));
    // d = 32, no dropout: the products start from -D_1 held in 16 registers and give G - D_1 at once; map 2 takes D_2 - D_1 off it (24 sequences
    // to 509: 79.4 us against 80.5; with d = 64 the registers are short: 16 x 178 16.6 against 16.2)
    constexpr bool HELD = D == 32 && !DROP;
    f32x16 nD;
    if constexpr (HELD) {
#pragma unroll
        for (int r = 0; r < 16; ++r) nD[r] = -Dq[0];
        asm volatile("" : "+v"(nD));                           // (registers, not 16 moves in every block)
        Dq[1] -= Dq[0];
    }
    if (nt > 0) kt.finish(0);
    else dma_wait();

    for (int t = 0; t < nt; ++t) {
        const bool general = kt.mk.general, none = kt.mk.out == ~0ull;
        if (t + 1 < nt) kt.start(t + 1);
        const bf16_t *Kt = kt.Kb(t), *Vt = kt.Vb(t);
        const int subs = none || idle ? 0 : min(2, (sk.n - t * KT + 31) >> 5);
        for (int u = 0; u < subs; ++u) {
            f32x16 g = HELD ? nD : zero16(), s[2];
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                s[j] = zero16();
#pragma unroll
                for (int ks = 0; ks < NS; ++ks)
                    s[j] = mfma32(row_frag<W>(Kt, u * 32 + (lane & 31), (j * D + ks * 16) / 8 + half), qf[j][ks], s[j]);
            }
#pragma unroll
            for (int i = 0; i < W / 16; ++i) g = mfma32(row_frag<W>(Vt, u * 32 + (lane & 31), 2 * i + half), gf[i], g);
            // weights 2^(s se - c): with a mask the maximum is taken off the masked score first, as in the forward pass
            float se = p.sc, c[2] = {c_lse[0], c_lse[1]};
            if (general) {
                se = 1.f;
#pragma unroll
                for (int j = 0; j < 2; ++j) c[j] = ll[j];
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const f32x4 mv = *reinterpret_cast<const f32x4*>(kt.Mb(t) + u * 32 + 8 * i + 4 * half);
#pragma unroll
                    for (int j = 0; j < 2; ++j)
#pragma unroll
                        for (int e = 0; e < 4; ++e) s[j][4 * i + e] = __builtin_fmaf(s[j][4 * i + e], p.sc, mv[e]) - m[j];
                }
            }
            if constexpr (DROP) {
                const Fields fl = fields16(p, drow, t * KT + u * 32, half);
#pragma unroll
                for (int r = 0; r < 16; ++r) g[r] = kept(p, fl, r) ? g[r] : 0.f;
            }
            bf16x8 df[2][2];
#pragma unroll
            for (int j = 0; j < 2; ++j) {
#pragma unroll
                for (int r = 0; r < 16; ++r) s[j][r] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[j][r], se, -c[j])) * (HELD && j == 0 ? g[r] : g[r] - Dq[j]);
                df[j][0] = pack_step(s[j], 0);
                df[j][1] = pack_step(s[j], 1);
            }
#pragma unroll
            for (int j = 0; j < 2; ++j)
#pragma unroll
                for (int t2 = 0; t2 < ND; ++t2)
#pragma unroll
                    for (int kk = 0; kk < 2; ++kk)
                        dq[j][t2] = mfma32(tr_frag<W>(Kt, u * 32 + kk * 16, j * D + t2 * 32, lane), df[j][kk], dq[j][t2]);
        }
        if (t + 1 < nt) kt.finish(t + 1);
    }
    const float z = p.sc * (1.f / LOG2E) * dscale;
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
// per query of a tile: max and log2(sum) of both maps, their sums, and D of both maps
enum { ST_M = 0, ST_LL = 2, ST_LSE = 4, ST_D = 6, ST_N = 8 };            // (ST_D without dropout: -D_1 and D_2 - D_1)

template <int D, bool DROP>
__device__ __forceinline__ void bwd_dkv_block(const DiffArgs& p, const Div nkb, const int bid, char* smem) {
    constexpr int W = 2 * D, NS = D / 16, ND = D / 32, NV = W / 32;
    bf16_t *Qs = reinterpret_cast<bf16_t*>(smem), *Os = Qs + 2 * KT * W;
    float(*st)[ST_N][KT] = reinterpret_cast<float(*)[ST_N][KT]>(Os + 2 * KT * W);
    const int bh = over(bid, nkb), kb = bid - bh * (int)nkb.d;
    const int b = over(bh, p.by_heads), h = bh - b * p.heads;
    const Span sq = span_of(p.cu_q, p.tot_q, b, p.Lq), sk = span_of(p.cu_k, p.tot_k, b, p.Lk);
    const int lane = threadIdx.x & 63, wid = __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6)), half = lane >> 5;
    const int nw = (int)blockDim.x >> 6;
    if (kb * nw * 32 >= sk.n) return;
    const int kbase = (kb * nw + wid) * 32, key = kbase + (lane & 31);
    const bool live = key < sk.n, idle = kbase >= sk.n;
    int nt = (sq.n + KT - 1) / KT;
    if (p.mask != nullptr) {                                   // a workgroup whose keys are all out (-inf) has nothing to sum
        const float* row = p.mask + (int64_t)b * p.lmask;
        bool any = false;
        for (int k = lane; k < nw * 32; k += 64) {
            const int at = kb * nw * 32 + k;
            any = any || (at < sk.n && row[at] != -INFINITY);
        }
        if (!__any(any)) nt = 0;
    }
    const bf16_t* Q = p.q + (int64_t)b * p.bq * (p.cu_q == nullptr) + sq.row * p.lq + h * W;
    const bf16_t* dO = p.dctx != nullptr ? p.dctx + ((p.cu_q != nullptr ? sq.row : (int64_t)b * p.Lq) * p.heads + h) * W
                                         : p.dout + (int64_t)b * p.bdo * (p.cu_q == nullptr) + sq.row * p.ldo + h * W;
    const int64_t ldO = p.dctx != nullptr ? (int64_t)p.heads * W : p.ldo;
    const float dscale = DROP ? p.drop.scale : 1.f, iscale = DROP ? 1.f / p.drop.scale : 1.f;       // (as in the dQ pass)
    f32x4 s4;
    float d0, d1;
    auto start = [&](const int t) {
        dma_tile<W>(Qs + (t & 1) * KT * W, Q, p.lq, t * KT, sq.n, wid, nw, lane);
        dma_tile<W>(Os + (t & 1) * KT * W, dO, ldO, t * KT, sq.n, wid, nw, lane);
        if (wid == 0) {
            const int64_t at = (int64_t)bh * p.Lq + min(t * KT + lane, sq.n - 1);
            s4 = *reinterpret_cast<const f32x4*>(p.stats + at * NSTAT);
            d0 = p.D[at * 2];
            d1 = p.D[at * 2 + 1];
        }
    };
    auto finish = [&](const int t) {
        dma_wait();
        if (wid == 0) {
            asm volatile("" : "+v"(s4), "+v"(d0), "+v"(d1));
            const bool in = t * KT + lane < sq.n;                              // behind the last query: P = 0
            float(*w)[KT] = st[t & 1];
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                w[ST_M + j][lane] = s4[2 * j];
                w[ST_LL + j][lane] = in ? s4[2 * j + 1] : INFINITY;
                w[ST_LSE + j][lane] = in ? s4[2 * j] + s4[2 * j + 1] : INFINITY;
            }
            w[ST_D][lane] = DROP ? d0 * iscale : -d0;
            w[ST_D + 1][lane] = DROP ? d1 * iscale : d1 - d0;
        }
        __syncthreads();
    };
    if (nt > 0) start(0);

    // keys that are out for good (-inf) and lanes behind the end: zeros and P = 0, whatever stands there
    float mk = -INFINITY;
    if (live) mk = p.mask != nullptr ? mask_log2(p.mask[(int64_t)b * p.lmask + key]) : 0.f;
    const bool use = mk != -INFINITY, general = __any(mk != 0.f);
    const bf16_t* K = p.k + (int64_t)b * p.bk * (p.cu_k == nullptr) + (sk.row + min(key, sk.n - 1)) * p.lk + h * W + half * 8;
    const bf16_t* V = p.v + (int64_t)b * p.bv * (p.cu_k == nullptr) + (sk.row + min(key, sk.n - 1)) * p.lv + h * W + half * 8;
    bf16x8 kf[2][NS], vf[W / 16];
#pragma unroll
    for (int s = 0; s < W / 16; ++s) {
        const u32x4 a = ldg16<false>(K + s * 16), c = ldg16<false>(V + s * 16), none = {0u, 0u, 0u, 0u};
        kf[s / NS][s % NS] = __builtin_bit_cast(bf16x8, use ? a : none);
        vf[s] = __builtin_bit_cast(bf16x8, use ? c : none);
    }
    float e1, e2;
    lambda_of<D>(p, h, lane, e1, e2);
    const float lam = e1 - e2 + p.lambda_init;

    f32x16 dk[2][ND], dv[NV];
#pragma unroll
    for (int t = 0; t < NV; ++t) dv[t] = zero16();
#pragma unroll
    for (int j = 0; j < 2; ++j)
#pragma unroll
        for (int t = 0; t < ND; ++t) dk[j][t] = zero16();
    pin(kf[0]);
    pin(kf[1]);
    pin(vf);
    if (nt > 0) finish(0);

    for (int t = 0; t < nt; ++t) {
        if (t + 1 < nt) start(t + 1);
        const bf16_t* Qt = Qs + (t & 1) * KT * W;
        const bf16_t* Ot = Os + (t & 1) * KT * W;
        const int subs = idle ? 0 : min(2, (sq.n - t * KT + 31) >> 5);
        for (int u = 0; u < subs; ++u) {
            const float* w = &st[t & 1][0][u * 32 + 4 * half];
            f32x16 g = zero16(), s[2], a;
            if constexpr (!DROP)                               // the products give G - D_1 at once; map 2 takes D_2 - D_1 off it
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const f32x4 D4 = *reinterpret_cast<const f32x4*>(w + ST_D * KT + 8 * i);
#pragma unroll
                    for (int e = 0; e < 4; ++e) g[4 * i + e] = D4[e];
                }
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                s[j] = zero16();
#pragma unroll
                for (int ks = 0; ks < NS; ++ks)
                    s[j] = mfma32(row_frag<W>(Qt, u * 32 + (lane & 31), (j * D + ks * 16) / 8 + half), kf[j][ks], s[j]);
            }
#pragma unroll
            for (int i = 0; i < W / 16; ++i) g = mfma32(row_frag<W>(Ot, u * 32 + (lane & 31), 2 * i + half), vf[i], g);
            float se = p.sc;
            const float* cs = w + ST_LSE * KT;
            if (general) {
                se = 1.f;
                cs = w + ST_LL * KT;
#pragma unroll
                for (int j = 0; j < 2; ++j)
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const f32x4 m4 = *reinterpret_cast<const f32x4*>(w + (ST_M + j) * KT + 8 * i);
#pragma unroll
                        for (int e = 0; e < 4; ++e) s[j][4 * i + e] = __builtin_fmaf(s[j][4 * i + e], p.sc, mk) - m4[e];
                    }
            }
            uint32_t keep = ~0u;
            if constexpr (DROP) {
                // the draws come with a query per lane; the ballot of bit r holds, for either half of the wave, one key over the queries
                const uint64_t drow = (uint64_t)bh * (uint64_t)p.Lq + (uint64_t)(t * KT + u * 32 + (lane & 31));
                const Fields fl = fields16(p, drow, kbase, half);
                const int kl = lane & 31, reg = 4 * (kl >> 3) + (kl & 3), kh = (kl >> 2) & 1;
#pragma unroll
                for (int r = 0; r < 16; ++r) {
                    const unsigned long long bal = __ballot(kept(p, fl, r));
                    const uint32_t part = kh ? (uint32_t)(bal >> 32) : (uint32_t)bal;
                    keep = reg == r ? part : keep;                             // bit: query of this block
                }
#pragma unroll
                for (int r = 0; r < 16; ++r) g[r] = (keep >> (acc_row(r) + 4 * half)) & 1u ? g[r] : 0.f;
            }
#pragma unroll
            for (int j = 0; j < 2; ++j)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const f32x4 c4 = *reinterpret_cast<const f32x4*>(cs + j * KT + 8 * i);
                    const f32x4 D4 = *reinterpret_cast<const f32x4*>(w + (ST_D + j) * KT + 8 * i);
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const int r = 4 * i + e;
                        const float pr = __builtin_amdgcn_exp2f(__builtin_fmaf(s[j][r], se, -c4[e]));
                        a[r] = j == 0 ? pr : __builtin_fmaf(-lam, pr, a[r]);
                        s[j][r] = pr * (!DROP && j == 0 ? g[r] : g[r] - D4[e]);
                    }
                }
            if constexpr (DROP) {
#pragma unroll
                for (int r = 0; r < 16; ++r) a[r] = (keep >> (acc_row(r) + 4 * half)) & 1u ? a[r] : 0.f;
            }
#pragma unroll
            for (int kk = 0; kk < 2; ++kk) {
                const bf16x8 af = pack_step(a, kk);
#pragma unroll
                for (int t2 = 0; t2 < NV; ++t2) dv[t2] = mfma32(tr_frag<W>(Ot, u * 32 + kk * 16, t2 * 32, lane), af, dv[t2]);
#pragma unroll
                for (int j = 0; j < 2; ++j) {
                    const bf16x8 df = pack_step(s[j], kk);
#pragma unroll
                    for (int t2 = 0; t2 < ND; ++t2) dk[j][t2] = mfma32(tr_frag<W>(Qt, u * 32 + kk * 16, j * D + t2 * 32, lane), df, dk[j][t2]);
                }
            }
        }
        if (t + 1 < nt) finish(t + 1);
    }
    const float z = p.sc * (1.f / LOG2E) * dscale;
    bf16_t* dkp = p.dk + (int64_t)b * p.bdk * (p.cu_k == nullptr) + (sk.row + key) * p.ldk + h * W;
    bf16_t* dvp = p.dv + (int64_t)b * p.bdv * (p.cu_k == nullptr) + (sk.row + key) * p.ldv + h * W;
#pragma unroll
    for (int t = 0; t < NV; ++t) {
        if constexpr (DROP) dv[t] *= dscale;
        store_block32(dvp + t * 32, dv[t], half, live);
    }
#pragma unroll
    for (int j = 0; j < 2; ++j)
#pragma unroll
        for (int t = 0; t < ND; ++t) {
            dk[j][t] *= j == 0 ? z : -lam * z;
            store_block32(dkp + j * D + t * 32, dk[j][t], half, live);
        }
}

template <int D>
constexpr int bwd_lds() { return 4 * KT * 2 * D * 2 + 2 * ST_N * KT * 4; }     // the larger of the two: dK / dV
struct BwdGrid { Div nb, chunk; int total, blocks; };          // blocks of rows per (example, head); units per chunk; units; workgroups

// dQ; the sums of the parameters' gradients ride along behind its last workgroups
template <int D, bool DROP>
__global__ __launch_bounds__(256, 2) void diff_bwd_dq_kernel(const DiffArgs p, const ParamGrads g, const BwdGrid gq) {
    __shared__ __attribute__((aligned(16))) char smem[bwd_lds<D>()];
    warm_args<sizeof(DiffArgs) + sizeof(ParamGrads) + sizeof(BwdGrid)>();
    if ((int)blockIdx.x >= gq.blocks) return bwd_params_block<D>(p, g, (int)blockIdx.x - gq.blocks, reinterpret_cast<float*>(smem));
    const int bid = chunk_map((int)blockIdx.x, gq.chunk);
    if (bid < gq.total) bwd_dq_block<D, DROP>(p, gq.nb, bid, smem);
}
template <int D, bool DROP>
__global__ __launch_bounds__(256, 1) void diff_bwd_dkv_kernel(const DiffArgs p, const BwdGrid gk) {
    __shared__ __attribute__((aligned(16))) char smem[bwd_lds<D>()];
    warm_args<sizeof(DiffArgs) + sizeof(BwdGrid)>();
    const int bid = chunk_map((int)blockIdx.x, gk.chunk);
    if (bid < gk.total) bwd_dkv_block<D, DROP>(p, gk.nb, bid, smem);
}
// both, the longer work first
template <int D, bool DROP>
__global__ __launch_bounds__(256, 2) void diff_bwd_kernel(const DiffArgs p, const ParamGrads g, const BwdGrid gk, const BwdGrid gq) {
    __shared__ __attribute__((aligned(16))) char smem[bwd_lds<D>()];
    warm_args<sizeof(DiffArgs) + sizeof(ParamGrads) + 2 * sizeof(BwdGrid)>();
    int id = (int)blockIdx.x;
    if (id < gk.blocks) {
        const int bid = chunk_map(id, gk.chunk);
        if (bid < gk.total) bwd_dkv_block<D, DROP>(p, gk.nb, bid, smem);
        return;
    }
    id -= gk.blocks;
    if (id < gq.blocks) {
        const int bid = chunk_map(id, gq.chunk);
        if (bid < gq.total) bwd_dq_block<D, DROP>(p, gq.nb, bid, smem);
        return;
    }
    bwd_params_block<D>(p, g, id - gq.blocks, reinterpret_cast<float*>(smem));
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
    UH_CHECK_ARG(a->norm_weight == nullptr || a->norm_eps > 0.f, "norm_eps must be positive");
    UH_CHECK_ARG(a->q_row % 8 == 0 && a->k_row % 8 == 0 && a->v_row % 8 == 0 && a->q_batch % 8 == 0 && a->k_batch % 8 == 0 && a->v_batch % 8 == 0,
                 "row and batch strides must be multiples of 8 elements");
    UH_CHECK_ARG(a->q_row >= 0 && a->k_row >= 0 && a->v_row >= 0 && a->q_row < (1 << 24) && a->k_row < (1 << 24) && a->v_row < (1 << 24),
                 "row strides must be 0 .. 2^24 elements");
    UH_CHECK_ARG(aligned16(a->q) && aligned16(a->k) && aligned16(a->v) && aligned16(a->norm_weight), "q, k, v and norm_weight must be 16-byte aligned");
    UH_CHECK_ARG(a->lambda_q1 && a->lambda_k1 && a->lambda_q2 && a->lambda_k2, "null pointer");
    const int64_t blocks = a->B * a->heads * ((a->Lq > a->Lk ? a->Lq : a->Lk) / 32 + 1);
    UH_CHECK_ARG(blocks < ((int64_t)1 << 25), "too many tokens for one launch");           // (a launch has fewer than 2^32 threads)
    return 0;
}

// whether there are query / key rows at all
bool has_queries(const UniterDiffAttention* a) { return a->B > 0 && a->Lq > 0 && (a->cu_seqlens_q == nullptr || a->total_q > 0); }
bool has_keys(const UniterDiffAttention* a) { return a->B > 0 && a->Lk > 0 && (a->cu_seqlens_k == nullptr || a->total_k > 0); }

Div div_of(int64_t d) {
    Div v;
    v.d = (uint32_t)d;
    v.shift = 0;
    while (((int64_t)1 << v.shift) < d) ++v.shift;
    v.mul = (uint32_t)((((uint64_t)1 << 32) * (((uint64_t)1 << v.shift) - (uint64_t)d)) / (uint64_t)d + 1);
    return v;
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
    p.by_heads = div_of(p.heads); p.by_Lq = div_of(p.Lq > 0 ? p.Lq : 1);
    p.sc = LOG2E / sqrtf((float)a->head_dim);
    p.drop = make_dropout(a->p_drop, a->seed, a->offset);
    return p;
}

// Waves of 32 rows per workgroup, up to four.  (178 rows as 3 + 3 waves instead of 4 + 2 measured slower, d = 64 dK / dV 28.9 us against
// 24.0: a wave without rows still takes its share of the tile transfers.)
int waves_for(int64_t L) { return (int)(L >= 97 ? 4 : L < 1 ? 1 : (L + 31) / 32); }

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

// Splits of the keys in the forward pass.  Estimated time (us) of a launch whose fullest CU runs k workgroups side by side: tiles per
// workgroup, and two tiles' worth of prologue and epilogue, times the most of
//   one workgroup's own round (latency of its transfers and products):  2.0 (d = 32), 3.0 (d = 64)
//   its share of HBM where no other query block reads the same keys:   0.79 k, 1.58 k (16 / 32 KiB at 5.3 TB/s over 256 CUs)
//   the SIMDs' work:                                                   1.13, 1.85 per wave that shares one
// and joining costs a second launch and the partial sums' way to memory and back.  One query, keys out of memory (us): 4 x 12 heads, d = 32,
// 16381 keys: 16 splits (3 workgroups on every CU) 47, 20 50, 10 60; 8 x 8 heads, d = 64, 8192 keys: 8 splits 64, 16 68, 4 104; 6 heads,
// d = 64, 32768 keys: 85 splits 40, 64 41, 16 104.
int splits_for(const UniterDiffAttention* a) {
    const bool wide = a->head_dim == 64;
    const int nw = waves_for(a->Lq);
    const int64_t nqb = (a->Lq + 32 * nw - 1) / (32 * nw), wg = a->B * a->heads * nqb, nt = (a->Lk + KT - 1) / KT;
    const int side = wide ? 2 : nw == 4 ? 3 : 4;               // workgroups per CU: LDS (66 / 33 KiB), three waves per SIMD with d = 32
    const double alone = wide ? 3.0 : 2.0, simd = wide ? 1.85 : 1.13, hbm = (wide ? 1.58 : 0.79) / (double)nqb;
    const double part = (double)(a->B * a->heads * a->Lq) * (16.0 * a->head_dim + 16.0) * 2e-6 / 2.5;
    int best = 1;
    double cost = 1e30;
    for (int64_t ns = 1; ns <= 256 && ns <= nt && wg * ns <= 1024 + wg; ++ns) {
        const int64_t c = (wg * ns + 255) / 256;
        auto round = [&](int64_t k) { return fmax(alone, fmax(hbm * (double)k, simd * (double)((k * nw + 3) / 4))); };
        const double t = (double)((nt + ns - 1) / ns + 2) * ((double)(c / side) * round(side) + (c % side ? round(c % side) : 0.0)) + (ns > 1 ? 5.5 + (double)ns * part : 0.0);
        if (t < cost) { cost = t; best = (int)ns; }
    }
    return best;
}
size_t fwd_space(const UniterDiffAttention* a, int ns) {
    return ns > 1 ? (size_t)(a->B * a->heads * a->Lq) * ns * (NSTAT + 4 * a->head_dim) * 4 : 0;
}

// `per` units share operands; about 8 chunks or more for each XCD
struct Grid { unsigned blocks; int total, chunk; };
Grid grid_of(int64_t total, int per) {
    Grid g;
    g.total = (int)total;
    const int64_t c = total / 64;
    g.chunk = (int)(c < 1 ? 1 : c > per ? per : c);
    g.blocks = (unsigned)((total + 8 * g.chunk - 1) / (8 * g.chunk) * 8 * g.chunk);
    return g;
}

template <int D>
int launch_fwd(const DiffArgs& p, int ns, hipStream_t st) {
    const int nw = waves_for(p.Lq), nqb = (p.Lq + 32 * nw - 1) / (32 * nw);
    const Grid gr = grid_of((int64_t)p.B * p.heads * nqb * ns, nqb * ns);
    const dim3 grid(gr.blocks), block(64 * nw);
    const FwdGrid g{div_of(nqb), div_of(ns), div_of(gr.chunk), gr.total};
    const bool drop = p.drop.p > 0.f;
    if (ns > 1) {
        if (drop) hipLaunchKernelGGL((diff_fwd_kernel<D, true, true>), grid, block, 0, st, p, g);
        else hipLaunchKernelGGL((diff_fwd_kernel<D, false, true>), grid, block, 0, st, p, g);
        UH_LAUNCH_CHECK();
        const int64_t rows = (int64_t)p.B * p.heads * p.Lq;
        constexpr int NG = 64 / (2 * D / 8);                   // groups of lanes in a wave
        if (ns <= NG) hipLaunchKernelGGL((diff_join_kernel<D, 1>), dim3((unsigned)((rows + 4 * NG - 1) / (4 * NG))), dim3(256), 0, st, p, ns);
        else hipLaunchKernelGGL((diff_join_kernel<D, NG>), dim3((unsigned)((rows + 3) / 4)), dim3(256), 0, st, p, ns);
    } else {
        if (drop) hipLaunchKernelGGL((diff_fwd_kernel<D, true, false>), grid, block, 0, st, p, g);
        else hipLaunchKernelGGL((diff_fwd_kernel<D, false, false>), grid, block, 0, st, p, g);
    }
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
    const unsigned tail = (unsigned)(g.n_lam + (g.w != nullptr ? W / 8 : 0));
    auto plan = [&](int L, int nw) {
        const int nb = (L + 32 * nw - 1) / (32 * nw);
        const Grid gr = grid_of((int64_t)p.B * p.heads * nb, nb);
        return BwdGrid{div_of(nb > 0 ? nb : 1), div_of(gr.chunk), gr.total, (int)gr.blocks};
    };
    const bool drop = p.drop.p > 0.f;
    // d = 32: one launch for dQ and dK / dV, which fill the chip better together than one after the other (2048 tokens, whole backward pass:
    // 4 heads 76 us against 135, 16 heads 100 against 151, 64 heads 360 against 479).  d = 64: dK / dV needs a register budget of its own.
    if constexpr (D == 32) {
        const int nw = p.Lq > p.Lk ? waves_for(p.Lq) : waves_for(p.Lk);
        const BwdGrid gk = plan(p.Lk, nw), gq = plan(p.Lq, nw);
        const dim3 grid((unsigned)gk.blocks + (unsigned)gq.blocks + tail), block(64 * nw);
        if (drop) hipLaunchKernelGGL((diff_bwd_kernel<D, true>), grid, block, 0, st, p, g, gk, gq);
        else hipLaunchKernelGGL((diff_bwd_kernel<D, false>), grid, block, 0, st, p, g, gk, gq);
        UH_LAUNCH_CHECK();
    } else {
        const int nwq = waves_for(p.Lq), nwk = waves_for(p.Lk);
        const BwdGrid gq = plan(p.Lq, nwq), gk = plan(p.Lk, nwk);
        if (gk.blocks > 0) {
            if (drop) hipLaunchKernelGGL((diff_bwd_dkv_kernel<D, true>), dim3((unsigned)gk.blocks), dim3(64 * nwk), 0, st, p, gk);
            else hipLaunchKernelGGL((diff_bwd_dkv_kernel<D, false>), dim3((unsigned)gk.blocks), dim3(64 * nwk), 0, st, p, gk);
            UH_LAUNCH_CHECK();
        }
        const dim3 grid((unsigned)gq.blocks + tail), block(64 * nwq);
        if (drop) hipLaunchKernelGGL((diff_bwd_dq_kernel<D, true>), grid, block, 0, st, p, g, gq);
        else hipLaunchKernelGGL((diff_bwd_dq_kernel<D, false>), grid, block, 0, st, p, g, gq);
        UH_LAUNCH_CHECK();
    }
    return 0;
}

}  // namespace

extern "C" {

size_t uniter_diff_attention_fwd_workspace_bytes(const UniterDiffAttention* a) {
    return check(a) || !has_queries(a) ? 0 : fwd_space(a, splits_for(a));
}

int uniter_diff_attention_fwd(const UniterDiffAttention* a, void* out, int64_t out_row, int64_t out_batch, float* stats, float* maps,
                              void* workspace, size_t workspace_bytes, void* stream) {
    if (const int rc = check(a)) return rc;
    if (!has_queries(a)) return 0;
    UH_CHECK_ARG(a->q && out && (!has_keys(a) || (a->k && a->v)), "null pointer");
    UH_CHECK_ARG(aligned16(out) && aligned16(stats) && aligned16(maps), "out, stats and maps must be 16-byte aligned");
    UH_CHECK_ARG(out_row % 8 == 0 && out_batch % 8 == 0, "row and batch strides must be multiples of 8 elements");
    UH_CHECK_ARG((stats == nullptr) == (maps == nullptr), "stats and maps are kept together, or neither");
    DiffArgs p = args_of(a);
    p.out = (bf16_t*)out; p.lo = out_row; p.bo = out_batch;
    p.stats = stats; p.maps = maps;
    const int ns = splits_for(a);
    UH_CHECK_ARG(workspace_bytes >= fwd_space(a, ns) && (workspace != nullptr || ns == 1), "workspace too small");
    UH_CHECK_ARG(aligned16(workspace), "workspace must be 16-byte aligned");
    p.psum = (float*)workspace;
    p.pacc = (float*)workspace + (size_t)(a->B * a->heads * a->Lq) * ns * NSTAT;
    return a->head_dim == 32 ? launch_fwd<32>(p, ns, (hipStream_t)stream) : launch_fwd<64>(p, ns, (hipStream_t)stream);
}

size_t uniter_diff_attention_bwd_workspace_bytes(const UniterDiffAttention* a) { return check(a) ? 0 : bwd_space(a).bytes; }

int uniter_diff_attention_bwd(const UniterDiffAttention* a, const float* stats, const float* maps, const void* dout, int64_t dout_row,
                              int64_t dout_batch, const UniterDiffAttentionGrads* g, void* workspace, size_t workspace_bytes, void* stream) {
    if (const int rc = check(a)) return rc;
    UH_CHECK_ARG(g != nullptr, "null pointer");
    UH_CHECK_ARG((a->norm_weight != nullptr) || g->norm_weight == nullptr, "a gradient of norm_weight needs norm_weight");
    UH_CHECK_ARG(!has_queries(a) || (a->q && stats && maps && dout && g->q), "null pointer");
    UH_CHECK_ARG(!has_keys(a) || (a->k && a->v && g->k && g->v), "null pointer");
    UH_CHECK_ARG(aligned16(stats) && aligned16(maps) && aligned16(dout) && aligned16(g->q) && aligned16(g->k) && aligned16(g->v) && aligned16(workspace),
                 "tensors must be 16-byte aligned");
    UH_CHECK_ARG(dout_row >= 0 && dout_row < (1 << 24), "row strides must be 0 .. 2^24 elements");
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
