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
};

template <typename TX> struct XFrag;
template <> struct XFrag<bf16_t> {
    static constexpr int P = 1;
    bf16x8 p[1];
    __device__ __forceinline__ void load(const bf16_t* x, int n, bool vec) {          // n: how many of the eight exist
        if (vec && n >= 8) { p[0] = *(const bf16x8*)x; return; }
#pragma unroll
        for (int j = 0; j < 8; ++j) p[0][j] = j < n ? x[j] : (bf16_t)0.f;
    }
    __device__ __forceinline__ bf16x8 piece(int) const { return p[0]; }
};
// fp32 activations are the exact sum of three bf16 values (8 + 8 + 8 bits of significand, each cut off, not rounded)
template <> struct XFrag<float> {
    static constexpr int P = 3;
    float v[8];
    __device__ __forceinline__ void load(const float* x, int n, bool vec) {
        if (vec && n >= 8) {
            const f32x4 a = *(const f32x4*)x, b = *(const f32x4*)(x + 4);
#pragma unroll
            for (int j = 0; j < 4; ++j) { v[j] = a[j]; v[4 + j] = b[j]; }
            return;
        }
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] = j < n ? x[j] : 0.f;
    }
    static __device__ __forceinline__ float cut(float a) { return __builtin_bit_cast(float, __builtin_bit_cast(unsigned, a) & 0xFFFF0000u); }
    __device__ __forceinline__ bf16x8 piece(int i) const {
        u32x4 o;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            float a = v[2 * j], b = v[2 * j + 1];
            for (int q = 0; q < i; ++q) { a -= cut(a); b -= cut(b); }
            o[j] = __builtin_amdgcn_perm(__builtin_bit_cast(unsigned, b), __builtin_bit_cast(unsigned, a), 0x07060302u);
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

// NT tiles of 16 weight rows, MT tiles of 16 activation rows; GS: 32-column steps of a scale group (1, 2, 4).
// The waves of a workgroup take the 128-column chunks in turn and are added up through LDS.
#define W4_MAX_WAVES 8
template <typename TX, int GS, int MT, int NT>
__global__ __launch_bounds__(64 * W4_MAX_WAVES) void w4_matmul_kernel(W4Args a) {
    extern __shared__ f32x4 s_part[];                            // [waves][NT * MT][64]
    constexpr int NG = 4 / GS;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), waves = blockDim.x >> 6;
    const int i = lane & 15, g = lane >> 4;
    const int t0 = blockIdx.x * NT, m0 = blockIdx.y * 16 * MT;
    f32x4 tot[NT][MT];
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int m = 0; m < MT; ++m) tot[n][m] = (f32x4){0.f, 0.f, 0.f, 0.f};
    struct Stage { u32x4 w[NT]; bf16x4 sc[NT][NG]; XFrag<TX> x[MT][4]; };
    auto load = [&](Stage& st, int c) {
#pragma unroll
        for (int n = 0; n < NT; ++n) {
            const long t = min(t0 + n, a.tiles - 1);
            st.w[n] = a.w[(t * a.chunks + c) * 64 + lane];
#pragma unroll
            for (int q = 0; q < NG; ++q) st.sc[n][q] = *(const bf16x4*)(a.scales + ((t * a.chunks + c) * NG + q) * 16 + 4 * g);
        }
#pragma unroll
        for (int m = 0; m < MT; ++m) {
            const int row = m0 + 16 * m + i;
#pragma unroll
            for (int s = 0; s < 4; ++s) {
                const int k = c * 128 + 32 * s + 8 * g;
                const int n = row < a.M ? a.K - k : 0;
                st.x[m][s].load((const TX*)a.x + (n > 0 ? row * a.ldx + k : 0), n, a.vec_x);
            }
        }
    };
    auto compute = [&](const Stage& st) {
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
                f32x4 base = (f32x4){0.f, 0.f, 0.f, 0.f};
                bf16x8 xs[GS][XFrag<TX>::P];
#pragma unroll
                for (int s = 0; s < GS; ++s)
#pragma unroll
                    for (int p = 0; p < XFrag<TX>::P; ++p) {
                        xs[s][p] = st.x[m][q * GS + s].piece(p);
                        base = __builtin_amdgcn_mfma_f32_16x16x32_bf16(minus, xs[s][p], base, 0, 0, 0);
                    }
#pragma unroll
                for (int n = 0; n < NT; ++n) {
                    f32x4 acc = base;
#pragma unroll
                    for (int s = 0; s < GS; ++s)
#pragma unroll
                        for (int p = 0; p < XFrag<TX>::P; ++p) acc = __builtin_amdgcn_mfma_f32_16x16x32_bf16(wo[n][s], xs[s][p], acc, 0, 0, 0);
#pragma unroll
                    for (int r = 0; r < 4; ++r) tot[n][m][r] = fmaf(sc[n][r], acc[r], tot[n][m][r]);
                }
            }
        }
    };
    Stage st[2];
    if (wave < a.chunks) load(st[0], wave);
    for (int c = wave; c < a.chunks; c += 2 * waves) {
        if (c + waves < a.chunks) load(st[1], c + waves);
        compute(st[0]);
        if (c + waves < a.chunks) {
            if (c + 2 * waves < a.chunks) load(st[0], c + 2 * waves);
            compute(st[1]);
        }
    }
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int m = 0; m < MT; ++m) s_part[(wave * (NT * MT) + n * MT + m) * 64 + lane] = tot[n][m];
    __syncthreads();
    for (int j = threadIdx.x; j < NT * MT * 64; j += blockDim.x) {
        f32x4 v = s_part[j];
        for (int u = 1; u < waves; ++u) v += s_part[u * (NT * MT * 64) + j];
        const int nm = j >> 6, l = j & 63;
        const int row = m0 + 16 * (nm % MT) + (l & 15), n0 = (t0 + nm / MT) * 16 + 4 * (l >> 4);
        if (row >= a.M || n0 >= a.N) continue;
        const int cnt = min(4, a.N - n0);
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
}

template <typename TX, int GS>
static int launch_w4(hipStream_t s, const W4Args& a) {
    const int mt = a.M <= 16 ? 1 : a.M <= 32 ? 2 : 4;
    const int nt = a.tiles >= 1024 ? 2 : 1;
    const int waves = a.chunks >= 8 ? 8 : 4;
    const dim3 grid((a.tiles + nt - 1) / nt, (a.M + 16 * mt - 1) / (16 * mt)), block(64 * waves);
    const int lds = waves * nt * mt * 64 * 16;
#define L(MT, NT) hipLaunchKernelGGL((w4_matmul_kernel<TX, GS, MT, NT>), grid, block, lds, s, a)
    if (nt == 1) { if (mt == 1) L(1, 1); else if (mt == 2) L(2, 1); else L(4, 1); }
    else { if (mt == 1) L(1, 2); else if (mt == 2) L(2, 2); else L(4, 2); }
#undef L
    return avsr_launch_status();
}

extern "C" int avsr_w4_matmul(avsr_stream_t stream, int x_dtype, int out_dtype, const void* x, int64_t ldx, const void* packed,
                              const void* scales, int64_t group, const float* bias, int act, const void* residual, int64_t ldr,
                              void* y, int64_t ldy, int64_t M, int64_t N, int64_t K) {
    if (!x || !packed || !scales || !y || M < 0 || N <= 0 || K <= 0 || ldx < K || ldy < N || (residual && ldr < N)) return AVSR_EINVAL;
    if ((x_dtype != AVSR_F32 && x_dtype != AVSR_BF16) || (out_dtype != AVSR_F32 && out_dtype != AVSR_BF16)) return AVSR_EINVAL;
    if (act != AVSR_ACT_NONE && act != AVSR_ACT_GELU && act != AVSR_ACT_RELU) return AVSR_EINVAL;
    if (group != 32 && group != 64 && group != 128) return AVSR_EUNSUPPORTED;
    if (((uintptr_t)packed % 16) || ((uintptr_t)scales % 8) || N > (1LL << 28) || K > (1LL << 24) || M > (1 << 20)) return AVSR_EUNSUPPORTED;
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
