// Products of a few rows with 4-bit weights:  y[m,n] = act(sum_k x[m,k] w[n,k] + bias[n]) + residual[m,n],
// w[n,k] = (nibble - 8) * scale[n, k / group].
//
// The weights stream from HBM once; unpacking them has to keep up (two vector instructions per byte leave none to
// spare at 8 TB/s), and the multiplication is free: even one row fits a matrix instruction's 16 columns.  So the
// kernel puts the WEIGHTS on the rows of v_mfma_f32_16x16x32_bf16 and x on its columns.  A nibble q in mantissa bits
// 3..6 of the bf16 16.0 reads as 16 + q: one shift and one and-or make two operands.  The 24 too many are taken out by
// the accumulator: it starts a group as the product of -24 and x, computed by the same instruction, so that a group's
// sum comes out as sum (q - 8) x and is scaled in fp32.  All sums are fp32 (MFMA accumulators); an x that is not finite
// makes its row NaN, because -24 * inf and 16 * inf meet.
//
// Packed layout (words of eight nibbles): word[n/16][k/128][k/8 % 4][n % 16][k/32 % 4], nibble of k % 8 = e at bit
// 4*(e/2) + 16*(e%2): 16 bytes are what one lane needs for 128 columns of its row, a wave's load is 1 KiB in a row.
// Scales: bf16 [n/16][k/group][n % 16].
#include "common.h"

struct W4Args {
    const u32x4* w; const bf16_t* scales; const void* x; long ldx; const float* bias; const void* residual; long ldr; void* y; long ldy;
    int M, N, K, chunks, tiles, act, out_f32, vec_x, vec_y;
    int kw, block;                 // staged kernel: ways that share the columns (a power of two), chunks of x in LDS at once
};

// Eight values of x as matrix operands: bf16 as it is, fp32 as the exact sum of three bf16 values (8 + 8 + 8 bits of
// significand, each cut off, not rounded).
template <typename TX> struct XFrag;
template <> struct XFrag<bf16_t> {
    static constexpr int P = 1;
    bf16x8 v;
    __device__ __forceinline__ void load(const bf16_t* x) { v = *(const bf16x8*)x; }
    __device__ __forceinline__ void load(const bf16_t* x, int n) {                    // the first n of the eight, wherever they stand
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] = j < n ? x[j] : (bf16_t)0.f;
    }
    __device__ __forceinline__ bf16x8 piece(int) const { return v; }
};
template <> struct XFrag<float> {
    static constexpr int P = 3;
    f32x4 a, b;
    __device__ __forceinline__ void load(const float* x) { a = *(const f32x4*)x; b = *(const f32x4*)(x + 4); }
    __device__ __forceinline__ void load(const float* x, int n) {
#pragma unroll
        for (int j = 0; j < 4; ++j) { a[j] = j < n ? x[j] : 0.f; b[j] = 4 + j < n ? x[4 + j] : 0.f; }
    }
    // what three cuts leave of an infinity is NaN, like the sums it goes into
    static __device__ __forceinline__ float cut(float f) { return __builtin_bit_cast(float, __builtin_bit_cast(unsigned, f) & 0xFFFF0000u); }
    __device__ __forceinline__ bf16x8 piece(int i) const {
        u32x4 o;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            float x = j < 2 ? a[2 * j] : b[2 * j - 4], y = j < 2 ? a[2 * j + 1] : b[2 * j - 3];
            for (int q = 0; q < i; ++q) { x -= cut(x); y -= cut(y); }
            o[j] = __builtin_amdgcn_perm(__builtin_bit_cast(unsigned, y), __builtin_bit_cast(unsigned, x), 0x07060302u);
        }
        return __builtin_bit_cast(bf16x8, o);
    }
};

__device__ __forceinline__ bf16x8 w4_operand(unsigned w) {      // 16 + nibble, in the order of k
    u32x4 o;
    o[0] = ((w << 3) & 0x00780078u) | 0x41804180u;
    o[1] = ((w >> 1) & 0x00780078u) | 0x41804180u;
    o[2] = ((w >> 5) & 0x00780078u) | 0x41804180u;
    o[3] = ((w >> 9) & 0x00780078u) | 0x41804180u;
    return __builtin_bit_cast(bf16x8, o);
}

// A wave's share: NT tiles of 16 weight rows times MT tiles of 16 rows of x; GS: 32-column steps of a scale group (1, 2, 4).
template <int GS, int MT, int NT> struct W4Wave {
    static constexpr int NG = 4 / GS;
    struct W { u32x4 w[NT]; bf16x4 sc[NT][NG]; };                // 128 columns of the weights
    const u32x4* wp[NT];
    const bf16_t* sp[NT];
    f32x4 tot[NT][MT];
    __device__ __forceinline__ W4Wave(const W4Args& a, int t0, int lane) {
#pragma unroll
        for (int n = 0; n < NT; ++n) {
            const long t = min(t0 + n, a.tiles - 1);             // a tile behind the last is computed like it and not stored
            wp[n] = a.w + t * a.chunks * 64 + lane;
            sp[n] = a.scales + t * a.chunks * NG * 16 + 4 * (lane >> 4);
#pragma unroll
            for (int m = 0; m < MT; ++m) tot[n][m] = (f32x4){0.f, 0.f, 0.f, 0.f};
        }
    }
    __device__ __forceinline__ void load(W& st, int c) const {
#pragma unroll
        for (int n = 0; n < NT; ++n) {
            st.w[n] = wp[n][c * 64];
#pragma unroll
            for (int q = 0; q < NG; ++q) st.sc[n][q] = *(const bf16x4*)(sp[n] + (c * NG + q) * 16);
        }
    }
    template <int P, typename X> __device__ __forceinline__ void add(const W& st, X x) {      // x(m, s, p): operand of step s, piece p
        bf16x8 minus;
#pragma unroll
        for (int j = 0; j < 8; ++j) minus[j] = (bf16_t)-24.f;
#pragma unroll
        for (int q = 0; q < NG; ++q) {
            bf16x8 wo[NT][GS];
            f32x4 sc[NT];
#pragma unroll
            for (int n = 0; n < NT; ++n) {
#pragma unroll
                for (int s = 0; s < GS; ++s) wo[n][s] = w4_operand(st.w[n][q * GS + s]);
#pragma unroll
                for (int r = 0; r < 4; ++r) sc[n][r] = (float)st.sc[n][q][r];
            }
#pragma unroll
            for (int m = 0; m < MT; ++m) {
                // each piece of x has sums of its own: within one, products have 16 bits and hardly any rounding takes place while
                // the 24 x come and go; the smaller pieces would be rounded at the largest one's 24 x
                f32x4 base[P], acc[NT][P];
                bf16x8 xs[GS][P];
#pragma unroll
                for (int p = 0; p < P; ++p) base[p] = (f32x4){0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int s = 0; s < GS; ++s)
#pragma unroll
                    for (int p = 0; p < P; ++p) {
                        xs[s][p] = x(m, q * GS + s, p);
                        base[p] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(minus, xs[s][p], base[p], 0, 0, 0);
                    }
#pragma unroll
                for (int n = 0; n < NT; ++n)
#pragma unroll
                    for (int p = 0; p < P; ++p) acc[n][p] = base[p];
#pragma unroll
                for (int s = 0; s < GS; ++s)
#pragma unroll
                    for (int p = 0; p < P; ++p)
#pragma unroll
                        for (int n = 0; n < NT; ++n) acc[n][p] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(wo[n][s], xs[s][p], acc[n][p], 0, 0, 0);
#pragma unroll
                for (int n = 0; n < NT; ++n)
#pragma unroll
                    for (int r = 0; r < 4; ++r) {
                        const float v = P == 1 ? acc[n][0][r] : acc[n][0][r] + (acc[n][1 % P][r] + acc[n][2 % P][r]);
                        tot[n][m][r] = fmaf(sc[n][r], v, tot[n][m][r]);
                    }
            }
        }
    }
    // The kw waves that share these tiles add up through LDS (room for all waves' sums); part p finishes every kw-th tile.
    __device__ __forceinline__ void finish(const W4Args& a, f32x4* sum, int t0, int m0, int wave, int part, int kw, int lane) {
        if (kw > 1) {
            __syncthreads();
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
                for (int m = 0; m < MT; ++m) sum[(wave * NT * MT + n * MT + m) * 64 + lane] = tot[n][m];
            __syncthreads();
        }
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int m = 0; m < MT; ++m) {
                if ((n * MT + m) % kw != part) continue;
                f32x4 v = tot[n][m];
                if (kw > 1) {
                    const f32x4* p = sum + ((wave - part) * NT * MT + n * MT + m) * 64 + lane;
                    v = p[0];
                    for (int u = 1; u < kw; ++u) v += p[u * NT * MT * 64];
                }
                store(a, v, m0 + 16 * m + (lane & 15), (t0 + n) * 16 + 4 * (lane >> 4));
            }
    }
    static __device__ __forceinline__ void store(const W4Args& a, f32x4 v, int row, int n0) {
        const int cnt = min(4, a.N - n0);
        if (row >= a.M || cnt <= 0) return;
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            if (r >= cnt) break;
            float z = v[r] + (a.bias ? a.bias[n0 + r] : 0.f);
            if (a.act == AVSR_ACT_GELU) z = gelu_erf(z);
            else if (a.act == AVSR_ACT_RELU) z = z < 0.f ? 0.f : z;
            if (a.residual) z += a.out_f32 ? ((const float*)a.residual)[row * a.ldr + n0 + r] : (float)((const bf16_t*)a.residual)[row * a.ldr + n0 + r];
            v[r] = z;
        }
        if (a.out_f32) {
            float* y = (float*)a.y + row * a.ldy + n0;
            if (a.vec_y && cnt == 4) *(f32x4*)y = v;
            else
                for (int r = 0; r < cnt; ++r) y[r] = v[r];
        } else {
            bf16_t* y = (bf16_t*)a.y + row * a.ldy + n0;
            if (a.vec_y && cnt == 4) {
                bf16x4 o;
#pragma unroll
                for (int r = 0; r < 4; ++r) o[r] = (bf16_t)v[r];
                *(bf16x4*)y = o;
            } else
                for (int r = 0; r < cnt; ++r) y[r] = (bf16_t)v[r];
        }
    }
};

// ---- x straight from L2: nothing to wait for before the first product.  1x16384x8192 (69 MB) takes 16 us, 4.3 TB/s, of
// which 12 are the bytes at the rate of a long read; a layer of a small decoder (1x1152x384) 3.5 us, a launch and two trips
// to memory.  Up to 16 rows.  The waves of a workgroup take the 128-column chunks in turn.  A chunk's weights and scales
// (AHEAD: its x too) are loaded while the one before is multiplied.  Rows of x behind the last are read as the last one: their
// columns of the product are never stored.
#define W4_WAVES 8
template <typename TX, int GS, int NT, bool AHEAD>
__global__ __launch_bounds__(64 * W4_WAVES) void w4_direct_kernel(W4Args a) {
    extern __shared__ f32x4 sums[];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), waves = blockDim.x >> 6;
    const int t0 = blockIdx.x * NT, g = lane >> 4;
    W4Wave<GS, 1, NT> ww(a, t0, lane);
    const TX* xp = (const TX*)a.x + (long)min(lane & 15, a.M - 1) * a.ldx + 8 * g;
    struct X { XFrag<TX> x[4]; };
    const int whole = a.vec_x ? a.K >> 7 : 0;                     // chunks whose x can be read in 16-byte pieces
    auto load_x = [&](X& st, int c) {
#pragma unroll
        for (int s = 0; s < 4; ++s) {
            const int k = c * 128 + 32 * s;
            if (c < whole) st.x[s].load(xp + k);
            else st.x[s].load(xp + k, a.K - (k + 8 * g));
        }
    };
    typename W4Wave<GS, 1, NT>::W sw[2];
    X sx[AHEAD ? 2 : 1];
    auto add = [&](int u) {
        const X& x = sx[AHEAD ? u : 0];
        ww.template add<XFrag<TX>::P>(sw[u], [&](int, int s, int p) { return x.x[s].piece(p); });
    };
    // loads come back in order: x of a chunk is asked for before weights that are further ahead
    if (AHEAD && wave < a.chunks) load_x(sx[0], wave);
    if (wave < a.chunks) ww.load(sw[0], wave);
    for (int c0 = wave; c0 < a.chunks; c0 += 2 * waves) {
#pragma unroll
        for (int u = 0; u < 2; ++u) {
            const int c = c0 + u * waves;
            if (c >= a.chunks) break;
            if (!AHEAD) load_x(sx[0], c);
            if (c + waves < a.chunks) {
                if (AHEAD) load_x(sx[AHEAD ? u ^ 1 : 0], c + waves);
                ww.load(sw[u ^ 1], c + waves);
            }
            add(u);
        }
    }
    ww.finish(a, sums, t0, 0, wave, wave, waves, lane);
}

// ---- x through LDS, for more than a few rows.  A fragment of x is 16 rows: read from L2 it touches 16 cache lines per quarter of a
// wave, 64 lines for the 1 KiB of weights it is multiplied with, and every wave does so for its own columns.  Here eight waves
// share x, whose rows are read in order, and fp32 is taken apart once.  The waves are kw ways of the chunks times 8 / kw groups
// of weight tiles.  x is staged in blocks of chunks, as many as fit, a row 16 bytes longer than its values so that the 16 rows a
// fragment reads lie in different banks.  16x51865x1280 14 us (39 MB; 7 at the rate of a long read, the rest is filling the
// pipeline: a wave has ten chunks), 64x51865x768 22 us (direct 40), 64x5120x1280 7.9 us (direct 14.7; 3.3 MB of weights: staging x
// and two barriers are most of it), 64x8192x8192 35 us.
template <typename TX, int GS, int MT, int NT>
__global__ __launch_bounds__(64 * W4_WAVES, 4) void w4_staged_kernel(W4Args a) {
    extern __shared__ __attribute__((aligned(16))) char lds[];
    constexpr int P = XFrag<TX>::P;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int part = wave & (a.kw - 1), t0 = (blockIdx.x * (W4_WAVES / a.kw) + wave / a.kw) * NT, m0 = blockIdx.y * 16 * MT;
    const int rows = min(16 * MT, a.M - m0), stride = a.block * 256 + 16;
    W4Wave<GS, MT, NT> ww(a, t0, lane);
    const char* xl[MT];                                          // rows behind the last are read as the last one
#pragma unroll
    for (int m = 0; m < MT; ++m) xl[m] = lds + min(16 * m + (lane & 15), rows - 1) * stride + 16 * (lane >> 4);
    typename W4Wave<GS, MT, NT>::W sw[2];
    for (int b0 = 0; b0 < a.chunks; b0 += a.block) {
        const int b1 = min(a.chunks, b0 + a.block), first = b0 + part;
        if (first < b1) ww.load(sw[0], first);
        if (b0) __syncthreads();                                 // the block before has been read
        const int pieces = (b1 - b0) * 16;                       // of eight values, of a row
        constexpr int U = P * MT == 1 ? 4 : 2;                   // pieces in flight per thread
        for (int j0 = threadIdx.x; j0 < rows * pieces; j0 += U * 64 * W4_WAVES) {
            XFrag<TX> f[U];
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const int j = j0 + u * 64 * W4_WAVES;
                if (j >= rows * pieces) break;
                const int row = j / pieces, k = b0 * 128 + (j - row * pieces) * 8;
                const TX* x = (const TX*)a.x + (long)(m0 + row) * a.ldx + (k < a.K ? k : 0);
                if (a.vec_x && k + 8 <= a.K) f[u].load(x);
                else f[u].load(x, a.K - k);
            }
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const int j = j0 + u * 64 * W4_WAVES;
                if (j >= rows * pieces) break;
                const int row = j / pieces;
#pragma unroll
                for (int p = 0; p < P; ++p) *(bf16x8*)(lds + (p * rows + row) * stride + (j - row * pieces) * 16) = f[u].piece(p);
            }
        }
        __syncthreads();
        for (int c0 = first; c0 < b1; c0 += 2 * a.kw) {
#pragma unroll
            for (int u = 0; u < 2; ++u) {
                const int c = c0 + u * a.kw;
                if (c >= b1) break;
                if (c + a.kw < b1) ww.load(sw[u ^ 1], c + a.kw);
                const int at = (c - b0) * 256;
                ww.template add<P>(sw[u], [&](int m, int s, int p) { return *(const bf16x8*)(xl[m] + p * rows * stride + at + s * 64); });
            }
        }
    }
    ww.finish(a, (f32x4*)lds, t0, m0, wave, part, a.kw, lane);
}

#define W4_FILL 4096            // waves that the chip is given: 16 per CU
#define W4_WIDE 1024            // tiles of weight rows (16384 rows) from which a wave takes two: 32768 rows for 4 8.7 us (one: 9.9), 12288 rows 6.1 (5.6)
#define W4_GROUPS 144           // workgroups of the staged kernel, at least: each of them reads all its rows of x, so not many more either
#define W4_X_BYTES 65536        // x in LDS where two workgroups share a CU; twice that where each has one to itself
template <typename TX, int GS>
static int launch_w4(hipStream_t s, W4Args a) {
    constexpr int P = XFrag<TX>::P, PAIR = P == 1 ? 2 : 1;        // two tiles for one read of x, registers permitting
    const bool wide = a.tiles >= W4_WIDE;
    // x goes through LDS above 16 rows (64x5120x1280 14.7 -> 7.9 us, 64x1280x5120 22 -> 11.6), in wide layers above 8 (51865x1280
    // for 16 14.1 us, direct 16.7; for 4 9.0 and 8.7).  At 16 rows of a layer that is not wide it is a matter of K: 16x5120x1280
    // 5.5 us, direct 6.0, but 16x1280x5120 10.1 and 8.5.
    if (a.M > (wide ? 8 : 16)) {
        // rows of x a workgroup takes: 16, or 32 where the weights are too many to come from a cache the second time
        // (64x51865x1280 29 us, 16 rows 36, 64 rows 32); fp32 has no registers for them (48x20000x2048 29 us, 43)
        const int mt = P == 1 && wide && a.M > 16 ? 2 : 1, rb = (a.M + 16 * mt - 1) / (16 * mt);
        const int nt = (long)(a.tiles + PAIR - 1) / PAIR * rb < W4_GROUPS ? 1 : PAIR;
        const int groups = (a.tiles + nt - 1) / nt, rows = a.M < 16 * mt ? a.M : 16 * mt;
        a.kw = 1;                                                // ways that share the chunks: as few as fill the chip
        while (a.kw < W4_WAVES && a.kw < a.chunks && (long)groups * rb * a.kw < W4_WAVES * W4_GROUPS) a.kw *= 2;
        const int tw = W4_WAVES / a.kw;
        const dim3 grid((groups + tw - 1) / tw, rb), block(64 * W4_WAVES);
        const int room = (long)grid.x * rb <= 256 ? 2 * W4_X_BYTES : W4_X_BYTES, most = (room / (rows * P) - 16) / 256;
        const int blocks = (a.chunks + most - 1) / most;
        a.block = (a.chunks + blocks - 1) / blocks;              // blocks of one size, and whole rounds of the ways
        if (blocks > 1 && most >= a.kw) {
            a.block = (a.block + a.kw - 1) / a.kw * a.kw;
            if (a.block > most) a.block = most / a.kw * a.kw;
        }
        const int xb = rows * P * (a.block * 256 + 16), sb = a.kw > 1 ? W4_WAVES * nt * mt * 1024 : 0, lds = xb > sb ? xb : sb;
#define L(MT, NT)                                                                                                        \
    do {                                                                                                                 \
        static avsr_dev_flags set;                                                                                       \
        if (lds > 65536 && !avsr_allow_lds((const void*)w4_staged_kernel<TX, GS, MT, NT>, 2 * W4_X_BYTES, set)) return AVSR_EHIP; \
        hipLaunchKernelGGL((w4_staged_kernel<TX, GS, MT, NT>), grid, block, lds, s, a);                                  \
    } while (0)
        if (mt == 2) L(PAIR, PAIR);
        else if (nt == 2) L(1, PAIR);
        else L(1, 1);
#undef L
        return avsr_launch_status();
    }
    const int nt = wide ? 2 : 1, groups = (a.tiles + nt - 1) / nt;
    int waves = W4_FILL / groups;                                // no more than there are chunks
    waves = waves < 1 ? 1 : waves > W4_WAVES ? W4_WAVES : waves;
    waves = waves < a.chunks ? waves : a.chunks;
    const dim3 grid(groups), block(64 * waves);
    const int lds = waves > 1 ? waves * nt * 1024 : 0;
    if (nt == 2) hipLaunchKernelGGL((w4_direct_kernel<TX, GS, 2, P == 1>), grid, block, lds, s, a);
    else hipLaunchKernelGGL((w4_direct_kernel<TX, GS, 1, true>), grid, block, lds, s, a);
    return avsr_launch_status();
}

extern "C" int avsr_w4_matmul(avsr_stream_t stream, int x_dtype, int out_dtype, const void* x, int64_t ldx, const void* packed,
                              const void* scales, int64_t group, const float* bias, int act, const void* residual, int64_t ldr,
                              void* y, int64_t ldy, int64_t M, int64_t N, int64_t K) {
    if (!x || !packed || !scales || !y || M < 0 || N <= 0 || K <= 0 || ldx < K || ldy < N || (residual && ldr < N)) return AVSR_EINVAL;
    if ((x_dtype != AVSR_F32 && x_dtype != AVSR_BF16) || (out_dtype != AVSR_F32 && out_dtype != AVSR_BF16)) return AVSR_EINVAL;
    if (act != AVSR_ACT_NONE && act != AVSR_ACT_GELU && act != AVSR_ACT_RELU) return AVSR_EINVAL;
    if (group != 32 && group != 64 && group != 128) return AVSR_EUNSUPPORTED;
    if (((uintptr_t)packed % 16) || ((uintptr_t)scales % 8) || N > (1LL << 28) || K > (1LL << 24) || M > (1 << 19)) return AVSR_EUNSUPPORTED;
    if (M == 0) return AVSR_OK;
    const int xs = x_dtype == AVSR_F32 ? 4 : 8;
    const bool of = out_dtype == AVSR_F32;
    W4Args a = {(const u32x4*)packed, (const bf16_t*)scales, x, ldx, bias, residual, ldr, y, ldy, (int)M, (int)N, (int)K, (int)((K + 127) / 128),
                (int)((N + 15) / 16), act, of, ldx % xs == 0 && (uintptr_t)x % 16 == 0, ldy % 4 == 0 && (uintptr_t)y % (of ? 16 : 8) == 0};
    hipStream_t s = (hipStream_t)stream;
#define G(TX) (group == 32 ? launch_w4<TX, 1>(s, a) : group == 64 ? launch_w4<TX, 2>(s, a) : launch_w4<TX, 4>(s, a))
    return x_dtype == AVSR_F32 ? G(float) : G(bf16_t);
#undef G
}
