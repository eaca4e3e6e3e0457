// Serving a decoder from a paged key / value cache.
//
//  * paged_plan_*_kernel: block tables, slot map and positions of one step from the requests' lengths, on the GPU.
//  * paged_write_kernel: the step's new keys and values into their slots.
//  * paged_attn_few_kernel / paged_attn_chunk_kernel: attention of the new tokens over the pages.
//
// A page holds `page` tokens of one layer: element (p, h, t, d) of the keys lives at K + p*sp + h*sh + t*D + d, the
// values in the same way (the [page, D] block of a page and head is contiguous, page and head strides are free).
#include "common.h"

#define LOG2E 1.4426950408889634f

// ================================================================= plan ====
// Exclusive sums over the requests of {pages taken, pages given back, new tokens} decide everything: request b takes
// the pages ring[(head + take_b + k) % n], k < need_b, gives its own to ring[(head + count + give_b + k) % n], and its
// new tokens are rows start_b .. of the step.  All output depends on the sums, so ONE workgroup makes them; what
// follows is independent per token and page.  A step of up to PLAN_THREADS requests and PLAN_ONE rows is latency only:
// the same workgroup writes it, a thread the tokens of its own request where there are one or two, a wave those of a
// longer prompt (8 requests 3.0 us, 512 with 64 prompts of up to 400 tokens 8.1 us; as two launches 12.4).  Above that the
// sums are made in passes and a second launch spreads the rows over the chip.
#define PLAN_THREADS 1024
#define PLAN_ONE 8192
#define PLAN_BIG (1 << 20)     // largest pool of the one-launch form: 1024 requests of no more pages each do not overflow, one with more fails

struct PlanArgs {
    const int* lens; const int* add; int* table; long ld_table; int width; int* ring; int n_pages; const int* pool;
    int* lens_out; int* pool_out; int B; int shift; int max_tokens; int* q_start; int* slots; int* positions; int* status;
    int* ws;                       // two-launch form: [3][B] old length, first page taken, first page given; [3] head, count, ok
};

// three inclusive scans over the wave
__device__ __forceinline__ void wave_scan3(int (&v)[3], int lane) {
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
        int u[3];
#pragma unroll
        for (int q = 0; q < 3; ++q) u[q] = __shfl_up(v[q], o);
#pragma unroll
        for (int q = 0; q < 3; ++q) v[q] += lane >= o ? u[q] : 0;
    }
}

// what request b asks for: v = {pages it takes, pages it gives back, new tokens}; bad: what cannot be
__device__ __forceinline__ void plan_request(const PlanArgs& a, int b, int& len, int& add, int (&v)[3], int& bad) {
    len = add = v[0] = v[1] = v[2] = 0;
    if (b >= a.B) return;
    len = a.lens[b];
    add = a.add[b];
    const long room = (long)a.width << a.shift;                        // < 2^31
    if (len < 0) { bad |= 8; return; }
    if (len > room || (add >= 0 && (long)len + add > room)) { bad |= 2; return; }
    const int up = (1 << a.shift) - 1, have = (int)(((long)len + up) >> a.shift);
    if (add < 0) { v[1] = have; return; }
    v[2] = add;
    v[0] = (int)(((long)len + add + up) >> a.shift) - have;
}
__device__ __forceinline__ int ring_at(const PlanArgs& a, int head, int k) {          // head + k < 2 n_pages
    const unsigned at = (unsigned)head + (unsigned)k;
    return (int)(at >= (unsigned)a.n_pages ? at - a.n_pages : at);
}
// token k of a request that held len tokens and takes its new pages from number `take` on
__device__ __forceinline__ void plan_token(const PlanArgs& a, const int* row, int len, int take, int head, int t, int k) {
    const int pos = len + k, j = pos >> a.shift, have = (len + (1 << a.shift) - 1) >> a.shift;
    const int p = j < have ? row[j] : a.ring[ring_at(a, head, take + j - have)];
    a.slots[t] = (p << a.shift) + (pos & ((1 << a.shift) - 1));
    a.positions[t] = pos;
}
// new table entries, or the ended request's pages into the ring, for j = first, first + step ...
__device__ __forceinline__ void plan_pages(const PlanArgs& a, int* row, int len, int add, int take, int give, int head, int count, int first, int step) {
    const int up = (1 << a.shift) - 1, have = (len + up) >> a.shift;
    if (add < 0)
        for (int j = first; j < have; j += step) a.ring[ring_at(a, head, count + give + j)] = row[j];
    else
        for (int j = have + first; j < (len + add + up) >> a.shift; j += step) row[j] = a.ring[ring_at(a, head, take + j - have)];
}

template <bool ONE>
__global__ __launch_bounds__(PLAN_THREADS) void paged_plan_sums_kernel(PlanArgs a) {
    __shared__ int part[3][16];
    __shared__ long red[3][16];
    __shared__ int s_bad, s_long;
    __shared__ int s_list[ONE ? PLAN_THREADS : 1][6];
    const int tid = threadIdx.x, lane = tid & 63, w = tid >> 6, waves = blockDim.x >> 6;
    const int head = a.pool[0], count = a.pool[1];
    int len, add, v[3], bad = (head < 0 || head >= a.n_pages || count < 0 || count > a.n_pages) ? 8 : 0;
    if (tid == 0) { s_bad = 0; s_long = 0; }
    int st = 0;
    if (!ONE) {                                                        // totals first: nothing is written unless the whole step fits
        long sum[3] = {0, 0, 0};
        for (int b = tid; b < a.B; b += PLAN_THREADS) {
            plan_request(a, b, len, add, v, bad);
#pragma unroll
            for (int q = 0; q < 3; ++q) sum[q] += v[q];
        }
        __syncthreads();
        if (bad) atomicOr(&s_bad, bad);
#pragma unroll
        for (int q = 0; q < 3; ++q) {
            for (int o = 32; o; o >>= 1) sum[q] += __shfl_xor(sum[q], o);
            if (lane == 0) red[q][w] = sum[q];
        }
        __syncthreads();
        long tot[3] = {0, 0, 0};
#pragma unroll
        for (int q = 0; q < 3; ++q)
            for (int i = 0; i < waves; ++i) tot[q] += red[q][i];
        st = s_bad | (tot[0] > count ? 1 : 0) | (tot[2] > a.max_tokens ? 4 : 0) | (tot[1] + count > a.n_pages ? 8 : 0);
    }
    int carry[3] = {0, 0, 0}, ex[3];
    const int passes = ONE ? 1 : (a.B + PLAN_THREADS - 1) / PLAN_THREADS;
    for (int c = 0; c < passes; ++c) {
        const int b = c * PLAN_THREADS + tid;
        plan_request(a, b, len, add, v, bad);
        int in[3];
#pragma unroll
        for (int q = 0; q < 3; ++q) {
            if (ONE) { if (v[q] > PLAN_BIG) bad |= 1 << 30; in[q] = min(v[q], PLAN_BIG); }
            else in[q] = st ? 0 : v[q];
            ex[q] = -in[q];
        }
        wave_scan3(in, lane);
        if (ONE) {
            for (int o = 1; o < 64; o <<= 1) bad |= __shfl_xor(bad, o);
            if (c == 0 && lane == 0) red[0][w] = bad;
        }
#pragma unroll
        for (int q = 0; q < 3; ++q)
            if (lane == 63) part[q][w] = in[q];
        __syncthreads();
#pragma unroll
        for (int q = 0; q < 3; ++q) {
            int base = carry[q], all = 0;
            for (int i = 0; i < waves; ++i) {
                const int u = part[q][i];
                base += i < w ? u : 0;
                all += u;
            }
            ex[q] += base + in[q];
            carry[q] += all;
        }
        if (ONE) {
            for (int i = 0; i < waves; ++i) st |= (int)red[0][i];
            if (st >> 30) {                                            // a request beyond any pool: the step fails, the status by exact sums
                long tot[3] = {0, 0, 0};
                int dummy = 0, l2, a2, v2[3];
                for (int i = 0; i < a.B; ++i) {
                    plan_request(a, i, l2, a2, v2, dummy);
#pragma unroll
                    for (int q = 0; q < 3; ++q) tot[q] += v2[q];
                }
                st &= ~(1 << 30);
                st |= (tot[0] > count ? 1 : 0) | (tot[2] > a.max_tokens ? 4 : 0) | (tot[1] + count > a.n_pages ? 8 : 0);
            } else st |= (carry[0] > count ? 1 : 0) | (carry[2] > a.max_tokens ? 4 : 0) | ((long)carry[1] + count > a.n_pages ? 8 : 0);
            if (st) carry[0] = carry[1] = carry[2] = ex[0] = ex[1] = ex[2] = 0;
        }
        if (b < a.B) {
            a.q_start[b] = ex[2];
            if (!ONE) { a.ws[b] = len; a.ws[a.B + b] = ex[0]; a.ws[2 * (long)a.B + b] = ex[1]; }
            if (!st) a.lens_out[b] = add < 0 ? 0 : len + add;
            else if (a.lens_out != a.lens) a.lens_out[b] = a.lens[b];
        }
        if (!ONE) __syncthreads();
    }
    if (tid == 0) {
        a.q_start[a.B] = carry[2];
        if (!ONE) { int* t = a.ws + 3 * (long)a.B; t[0] = head; t[1] = count; t[2] = !st; }
        a.status[0] = st;
        if (!st) {
            a.pool_out[0] = ring_at(a, head, carry[0]);
            a.pool_out[1] = count - carry[0] + carry[1];
        } else if (a.pool_out != a.pool) { a.pool_out[0] = head; a.pool_out[1] = count; }
    }
    if (!ONE) return;
    for (int t = carry[2] + tid; t < a.max_tokens; t += blockDim.x) { a.slots[t] = -1; a.positions[t] = 0; }
    if (st) return;
    if (tid < a.B) {
        int* row = a.table + tid * a.ld_table;
        if (v[2] <= 2 && v[0] <= 2 && v[1] <= 2) {
            for (int k = 0; k < v[2]; ++k) plan_token(a, row, len, ex[0], head, ex[2] + k, k);
            plan_pages(a, row, len, add, ex[0], ex[1], head, count, 0, 1);
        } else {
            int* e = s_list[atomicAdd(&s_long, 1)];
            e[0] = tid; e[1] = len; e[2] = add; e[3] = ex[0]; e[4] = ex[1]; e[5] = ex[2];
        }
    }
    __syncthreads();
    for (int i = w; i < s_long; i += waves) {
        const int* e = s_list[i];
        int* row = a.table + e[0] * a.ld_table;
        for (int k = lane; k < e[2]; k += 64) plan_token(a, row, e[1], e[3], head, e[5] + k, k);
        plan_pages(a, row, e[1], e[2], e[3], e[4], head, count, lane, 64);
    }
}
__global__ __launch_bounds__(256) void paged_plan_rows_kernel(PlanArgs a) {
    const int* s = a.ws + 3 * (long)a.B;
    const int head = s[0], count = s[1], total = a.q_start[a.B];
    const long tid = (long)blockIdx.x * 256 + threadIdx.x, nthr = (long)gridDim.x * 256;
    const int *len = a.ws, *take = a.ws + a.B, *give = a.ws + 2 * (long)a.B;
    for (long t = tid; t < a.max_tokens; t += nthr) {
        if (t >= total) { a.slots[t] = -1; a.positions[t] = 0; continue; }
        int lo = 0, hi = a.B;                                          // q_start[lo] <= t < q_start[hi]
        while (hi - lo > 1) {
            const int mid = (lo + hi) >> 1;
            if (a.q_start[mid] <= t) lo = mid; else hi = mid;
        }
        plan_token(a, a.table + lo * a.ld_table, len[lo], take[lo], head, (int)t, (int)t - a.q_start[lo]);
    }
    if (!s[2]) return;
    for (long b = tid >> 6; b < a.B; b += nthr >> 6)                   // a wave per request
        plan_pages(a, a.table + b * a.ld_table, len[b], a.add[b], take[b], give[b], head, count, (int)(tid & 63), 64);
}

static inline int page_shift(int64_t page) {
    for (int s = 4; s <= 8; ++s)
        if (page == (1 << s)) return s;
    return -1;
}
static inline bool plan_one(int64_t B, int64_t max_tokens, int64_t n_pages) { return B <= PLAN_THREADS && max_tokens <= PLAN_ONE && n_pages <= PLAN_BIG; }

extern "C" int64_t avsr_paged_plan_workspace_bytes(int64_t B, int64_t max_tokens, int64_t n_pages) {
    return plan_one(B, max_tokens, n_pages) ? 0 : (3 * B + 4) * 4;
}

extern "C" int avsr_paged_plan(avsr_stream_t stream, const int32_t* lens, const int32_t* add, int32_t* table, int64_t ld_table,
                               int64_t width, int32_t* ring, int64_t n_pages, const int32_t* pool, int64_t B, int64_t page,
                               int64_t max_tokens, int32_t* lens_out, int32_t* pool_out, int32_t* q_start, int32_t* slots,
                               int32_t* positions, int32_t* status, void* workspace) {
    if (!lens || !add || !table || !ring || !pool || !lens_out || !pool_out || !q_start || !slots || !positions || !status) return AVSR_EINVAL;
    if (B <= 0 || width <= 0 || ld_table < width || n_pages <= 0 || max_tokens <= 0) return AVSR_EINVAL;
    const int shift = page_shift(page);
    // slots, lengths and ring positions are 32-bit
    if (shift < 0 || B > (1 << 24) || max_tokens > (1 << 30) || n_pages > (1LL << (30 - shift)) || width > (1LL << (30 - shift))) return AVSR_EUNSUPPORTED;
    if (!plan_one(B, max_tokens, n_pages) && !workspace) return AVSR_EINVAL;
    PlanArgs a = {lens, add, table, (long)ld_table, (int)width, ring, (int)n_pages, pool, lens_out, pool_out, (int)B, shift, (int)max_tokens,
                  q_start, slots, positions, status, (int*)workspace};
    hipStream_t s = (hipStream_t)stream;
    if (plan_one(B, max_tokens, n_pages)) {
        // a thread per request, and enough for the rows to be done in a few turns
        const int64_t want = B > max_tokens / 4 ? B : max_tokens / 4;
        const int threads = want >= PLAN_THREADS ? PLAN_THREADS : (int)((want + 63) / 64 * 64);
        hipLaunchKernelGGL(paged_plan_sums_kernel<true>, dim3(1), dim3(threads), 0, s, a);
    } else {
        hipLaunchKernelGGL(paged_plan_sums_kernel<false>, dim3(1), dim3(PLAN_THREADS), 0, s, a);
        int64_t blocks = (max_tokens + 255) / 256, more = (B + 3) / 4;
        blocks = blocks > more ? blocks : more;
        hipLaunchKernelGGL(paged_plan_rows_kernel, dim3((unsigned)(blocks < 2048 ? blocks : 2048)), dim3(256), 0, s, a);
    }
    return avsr_launch_status();
}

// ================================================================ write ====
// One 16-byte piece of a page per thread and turn; a row of the pages (one token and head) is 128 or more contiguous
// bytes.  Pure traffic: every byte is read once and written once (48000 tokens of 20 heads, 492 MB, in 95 us: 5.2 TB/s, the
// rate of a large copy; 8 tokens 2.6 us).
template <typename TI, typename TO> struct WritePiece;
template <typename T> struct WritePiece<T, T> {
    static constexpr int N = 16 / sizeof(T);
    u32x4 v;
    __device__ void load(const T* p) { v = *(const u32x4*)p; }
    __device__ void store(T* p) const { *(u32x4*)p = v; }
};
template <> struct WritePiece<float, bf16_t> {
    static constexpr int N = 8;
    f32x4 a, b;
    __device__ void load(const float* p) { a = *(const f32x4*)p; b = *(const f32x4*)(p + 4); }
    __device__ void store(bf16_t* p) const {
        bf16x8 o;
#pragma unroll
        for (int i = 0; i < 4; ++i) { o[i] = (bf16_t)a[i]; o[4 + i] = (bf16_t)b[i]; }     // the cache's type: one rounding
        *(bf16x8*)p = o;
    }
};
struct WriteArgs {
    const void *k, *v; long ldk, ldv, hk, hv;          // token and head strides of the new rows
    void *kp, *vp; long sp, sh, svp, svh;
    const int* slots; long rows; int H, dshift, shift; long n_slots;
};
template <typename TI, typename TO, int U>
__global__ __launch_bounds__(256) void paged_write_kernel(WriteArgs a) {
    typedef WritePiece<TI, TO> P;
    const int per_row = 1 << (a.dshift - (P::N == 8 ? 3 : 2));          // pieces of one head
    const unsigned per_tok = 2u * a.H * per_row;
    const long n = a.rows * per_tok;
    const long first = (long)blockIdx.x * (256 * U) + threadIdx.x;
    P x[U];
    TO* dst[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
        dst[u] = nullptr;
        const long i = first + u * 256;
        if (i >= n) continue;
        const long t = n < (1L << 32) ? (long)((unsigned)i / per_tok) : i / per_tok;
        const int c = (int)(i - t * per_tok);
        const int slot = a.slots[t];
        if (slot < 0 || slot >= a.n_slots) continue;                    // no row to store, or no such page
        int h = c / per_row;
        const int d = (c - h * per_row) * P::N;
        const bool isv = h >= a.H;
        h -= isv ? a.H : 0;
        const long p = slot >> a.shift, off = slot & ((1 << a.shift) - 1);
        x[u].load((const TI*)(isv ? a.v : a.k) + t * (isv ? a.ldv : a.ldk) + h * (isv ? a.hv : a.hk) + d);
        dst[u] = (TO*)(isv ? a.vp : a.kp) + p * (isv ? a.svp : a.sp) + h * (isv ? a.svh : a.sh) + (off << a.dshift) + d;
    }
#pragma unroll
    for (int u = 0; u < U; ++u)
        if (dst[u]) x[u].store(dst[u]);
}

extern "C" int avsr_paged_write(avsr_stream_t stream, int in_dtype, int page_dtype, const void* k, int64_t ldk, int64_t k_head,
                                const void* v, int64_t ldv, int64_t v_head, void* k_pages, int64_t k_page_stride,
                                int64_t k_head_stride, void* v_pages, int64_t v_page_stride, int64_t v_head_stride,
                                const int32_t* slots, int64_t rows, int64_t H, int64_t head_dim, int64_t page, int64_t n_pages) {
    if (!k || !v || !k_pages || !v_pages || !slots || rows < 0 || H <= 0 || n_pages <= 0) return AVSR_EINVAL;
    const int shift = page_shift(page);
    if (shift < 0 || (head_dim != 64 && head_dim != 128) || n_pages > (1LL << (30 - shift)) || H > (1 << 16)) return AVSR_EUNSUPPORTED;
    const int64_t qi = in_dtype == AVSR_F32 ? 4 : 8, qo = page_dtype == AVSR_F32 ? 4 : 8;
    // the stride of a dimension of one is never used
    if (rows <= 1) ldk = ldv = 0;
    if (H == 1) k_head = v_head = k_head_stride = v_head_stride = 0;
    if (n_pages == 1) k_page_stride = v_page_stride = 0;
    if ((ldk | ldv | k_head | v_head) % qi || (k_page_stride | k_head_stride | v_page_stride | v_head_stride) % qo ||
        ((uintptr_t)k | (uintptr_t)v | (uintptr_t)k_pages | (uintptr_t)v_pages) % 16) return AVSR_EUNSUPPORTED;
    if (rows == 0) return AVSR_OK;
    WriteArgs a = {k, v, ldk, ldv, k_head, v_head, k_pages, v_pages, k_page_stride, k_head_stride, v_page_stride, v_head_stride,
                   slots, rows, (int)H, head_dim == 64 ? 6 : 7, shift, n_pages << shift};
    const int64_t n = rows * 2 * H * head_dim / ((in_dtype == AVSR_F32 && page_dtype == AVSR_F32) ? 4 : 8);
    hipStream_t s = (hipStream_t)stream;
    const int64_t blocks = (n + 1023) / 1024;
    if (blocks > 0xffffff) return AVSR_EUNSUPPORTED;             // a launch has fewer than 2^32 threads
#define L(TI, TO) hipLaunchKernelGGL((paged_write_kernel<TI, TO, 4>), dim3((unsigned)blocks), dim3(256), 0, s, a)
    if (in_dtype == AVSR_BF16 && page_dtype == AVSR_BF16) L(bf16_t, bf16_t);
    else if (in_dtype == AVSR_F32 && page_dtype == AVSR_F32) L(float, float);
    else if (in_dtype == AVSR_F32 && page_dtype == AVSR_BF16) L(float, bf16_t);
    else return AVSR_EINVAL;
#undef L
    return avsr_launch_status();
}

// ============================================================ attention ====
// Scores are made transposed, S^T = K.Q^T, with 16 query rows as the columns of the tile: a lane owns one row (column
// lane & 15), softmax statistics are per lane, and the S^T accumulator is, register for register, the B operand of
// O^T = V^T.P^T.  The order of the keys inside a tile of 32 is free, and chosen so that a lane's eight scores are eight
// neighbouring keys (bf16, key 8g + 4t + r of sub-tile t, register r, g = lane / 16): the A operand V^T then is eight
// key rows of one column, which the lane gets from whole 8- or 16-byte pieces of those rows by register permutes.
// Neither K nor V passes through LDS.
//
// Row r of a request's tile is query token r / G, query head hk*G + r % G of the G heads that share a kv head.
struct AttnArgs {
    const void* q; long ldq, hq;                  // token and head strides
    const void *k, *v; long sp, sh, svp, svh;
    const int* table; long ld_table; int width;
    const int* lens; const int* q_start;
    void* o; long ldo, ho;
    int B, Hk, G, N, shift, n_pages; float c; int causal;     // c = scale * log2(e)
    int splits, few_rows;                         // key splits; most rows of a request that the first kernel takes (0 = any)
    int n_few, few_tiles;                         // second kernel: workgroups in its grid that do the first one's work, tiles of 16 rows
    float *part, *part_ml;                        // [rows][splits][D] sums and [rows][splits]{m, l} of a split grid
};

// Rows, lengths of request b, kept inside what the arrays hold.
struct Req { int q0, nq, len; };
__device__ __forceinline__ Req request(const AttnArgs& a, int b) {
    Req r;
    const int s = a.q_start[b], e = a.q_start[b + 1];
    r.q0 = min(max(s, 0), a.N);
    r.nq = max(min(e, a.N) - r.q0, 0);
    r.len = min(max(a.lens[b], 0), a.width << a.shift);
    return r;
}

__device__ __forceinline__ bool finite(float f) { return (__builtin_bit_cast(unsigned, f) & 0x7F800000u) != 0x7F800000u; }
// the halves (bf16) of v whose exponent is all ones - infinities and NaN - cleared; odd: set if there were any
__device__ __forceinline__ unsigned finite_half(unsigned v, bool& odd) {
    const bool lo = (v & 0x7F80u) == 0x7F80u, hi = (v & 0x7F800000u) == 0x7F800000u;
    odd |= lo || hi;
    return v & ((lo ? 0u : 0xFFFFu) | (hi ? 0u : 0xFFFF0000u));
}

// Probabilities go into the second product as the sum of two bf16 values, the nearest one and the nearest to what is left: off by
// 2^-16 of themselves at most, so that a bf16 result is the exact one rounded once but for values next to a border (one value alone: 2^-8;
// against 64 bits 2.2e-3 of the result's norm where its own rounding is 1.66e-3).  The rest comes of one instruction, x - (hi . {1, 0}),
// exact because its bits are x's own.
struct Two { bf16x2 hi, lo; };
__device__ __forceinline__ Two two_pieces(float x, float y) {
    unsigned first = 0x0000BF80u, second = 0xBF800000u;               // {-1, 0} and {0, -1}; opaque: as an inline constant -1.0 has two meanings
    asm("" : "+s"(first), "+s"(second));
    Two t;
    t.hi = (bf16x2){(bf16_t)x, (bf16_t)y};
    t.lo = (bf16x2){(bf16_t)__builtin_amdgcn_fdot2_f32_bf16(t.hi, __builtin_bit_cast(bf16x2, first), x, false),
                    (bf16_t)__builtin_amdgcn_fdot2_f32_bf16(t.hi, __builtin_bit_cast(bf16x2, second), y, false)};
    return t;
}

template <typename T, int D> struct Frag;
// ---- bf16: v_mfma_f32_16x16x32_bf16 (A row / B column lane & 15, k = 8g + j; C column lane & 15, row 4g + r)
template <int D> struct Frag<bf16_t, D> {
    typedef bf16_t T;
    static constexpr int VW = D / 16;                                   // values of a key row per lane: columns VW*i ..
    typedef __attribute__((ext_vector_type(VW / 2))) unsigned vrow_t;
    struct Q { bf16x8 x[D / 32]; };
    struct K { bf16x8 x[2][D / 32]; };
    struct V { vrow_t x[8]; };
    static __device__ __forceinline__ int key_of_row(int t, int m) { return 8 * (m >> 2) + 4 * t + (m & 3); }
    static __device__ __forceinline__ int key_of_score(int t, int r, int g) { return 8 * g + 4 * t + r; }
    static __device__ __forceinline__ void load_q(Q& q, const T* p, int g, bool ok) {
#pragma unroll
        for (int c = 0; c < D / 32; ++c) {
            if (ok) q.x[c] = *(const bf16x8*)(p + 32 * c + 8 * g);
            else q.x[c] = (bf16x8){};
        }
    }
    // base0 / base1: the [page, D] block that holds keys 0..15 / 16..31 of the tile, already moved to the tile's first row of it
    static __device__ __forceinline__ void load_k(K& k, const T* base0, const T* base1, bool two, int i, int g) {
#pragma unroll
        for (int t = 0; t < 2; ++t) {
            const int key = key_of_row(t, i);
            const T* p = (two && (key & 16)) ? base1 + (key & 15) * D : base0 + key * D;
#pragma unroll
            for (int c = 0; c < D / 32; ++c) k.x[t][c] = *(const bf16x8*)(p + 32 * c + 8 * g);
        }
    }
    static __device__ __forceinline__ void load_v(V& v, const T* base0, const T* base1, bool two, int i, int g) {
        const T* p = ((two && g >= 2) ? base1 + (8 * g - 16) * D : base0 + 8 * g * D) + VW * i;
#pragma unroll
        for (int j = 0; j < 8; ++j) v.x[j] = *(const vrow_t*)(p + j * D);
    }
    static __device__ __forceinline__ void scores(f32x4 (&s)[2], const K& k, const Q& q) {
#pragma unroll
        for (int t = 0; t < 2; ++t) {
            s[t] = (f32x4){0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int c = 0; c < D / 32; ++c) s[t] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(k.x[t][c], q.x[c], s[t], 0, 0, 0);
        }
    }
    // column VW*i + e of the eight key rows, as an A operand
    static __device__ __forceinline__ bf16x8 column(const V& v, int e) {
        u32x4 f;
#pragma unroll
        for (int p = 0; p < 4; ++p)
            f[p] = __builtin_amdgcn_perm(v.x[2 * p + 1][e >> 1], v.x[2 * p][e >> 1], (e & 1) ? 0x07060302u : 0x05040100u);
        return __builtin_bit_cast(bf16x8, f);
    }
    static constexpr bool TWO = true;                                    // probabilities are two pieces
    struct P { bf16x8 hi, lo; };
    static __device__ __forceinline__ P probs(const f32x4 (&s)[2]) {
        P p;
#pragma unroll
        for (int r = 0; r < 8; r += 2) {
            const Two t = two_pieces(s[r >> 2][r & 3], s[r >> 2][(r & 3) + 1]);
            p.hi[r] = t.hi[0]; p.hi[r + 1] = t.hi[1];
            p.lo[r] = t.lo[0]; p.lo[r + 1] = t.lo[1];
        }
        return p;
    }
    static __device__ __forceinline__ void zero_key(V& v, int j) { v.x[j] = (vrow_t)(0u); }
    static __device__ __forceinline__ int key_of_v(int j, int g) { return 8 * g + j; }
    static __device__ __forceinline__ bool keep_finite(V& v) {           // clears what is not finite; whether there was any
        bool odd = false;
#pragma unroll
        for (int j = 0; j < 8; ++j)
#pragma unroll
            for (int w = 0; w < VW / 2; ++w) v.x[j][w] = finite_half(v.x[j][w], odd);
        return odd;
    }
    static __device__ __forceinline__ f32x4 pv(const V& v, int e, const P& p, f32x4 o) {
        const bf16x8 c = column(v, e);
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(c, p.hi, __builtin_amdgcn_mfma_f32_16x16x32_bf16(c, p.lo, o, 0, 0, 0), 0, 0, 0);
    }
};
// ---- fp32: v_mfma_f32_16x16x4_f32 (A row / B column lane & 15, k = g; C as above)
template <int D> struct Frag<float, D> {
    typedef float T;
    static constexpr int VW = D / 16;
    struct Q { f32x4 x[D / 16]; };
    struct K { f32x4 x[2][D / 16]; };
    struct V { f32x4 x[8][VW / 4]; };
    static __device__ __forceinline__ int key_of_row(int t, int m) { return 16 * t + m; }
    static __device__ __forceinline__ int key_of_score(int t, int r, int g) { return 16 * t + 4 * g + r; }
    static __device__ __forceinline__ void load_q(Q& q, const T* p, int g, bool ok) {
#pragma unroll
        for (int c = 0; c < D / 16; ++c) {
            if (ok) q.x[c] = *(const f32x4*)(p + 16 * c + 4 * g);
            else q.x[c] = (f32x4){0.f, 0.f, 0.f, 0.f};
        }
    }
    static __device__ __forceinline__ void load_k(K& k, const T* base0, const T* base1, bool two, int i, int g) {
#pragma unroll
        for (int t = 0; t < 2; ++t) {
            const T* p = (two && t) ? base1 + i * D : base0 + (16 * t + i) * D;
#pragma unroll
            for (int c = 0; c < D / 16; ++c) k.x[t][c] = *(const f32x4*)(p + 16 * c + 4 * g);
        }
    }
    static __device__ __forceinline__ void load_v(V& v, const T* base0, const T* base1, bool two, int i, int g) {
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const int t = j >> 2, k = 4 * g + (j & 3);
            const T* p = ((two && t) ? base1 + k * D : base0 + (16 * t + k) * D) + VW * i;
#pragma unroll
            for (int w = 0; w < VW / 4; ++w) v.x[j][w] = *(const f32x4*)(p + 4 * w);
        }
    }
    static __device__ __forceinline__ void scores(f32x4 (&s)[2], const K& k, const Q& q) {
#pragma unroll
        for (int t = 0; t < 2; ++t) {
            s[t] = (f32x4){0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int c = 0; c < D / 16; ++c)
#pragma unroll
                for (int x = 0; x < 4; ++x) s[t] = __builtin_amdgcn_mfma_f32_16x16x4f32(k.x[t][c][x], q.x[c][x], s[t], 0, 0, 0);
        }
    }
    static __device__ __forceinline__ void zero_key(V& v, int j) {
#pragma unroll
        for (int w = 0; w < VW / 4; ++w) v.x[j][w] = (f32x4){0.f, 0.f, 0.f, 0.f};
    }
    static __device__ __forceinline__ int key_of_v(int j, int g) { return 16 * (j >> 2) + 4 * g + (j & 3); }
    static __device__ __forceinline__ bool keep_finite(V& v) {
        bool odd = false;
#pragma unroll
        for (int j = 0; j < 8; ++j)
#pragma unroll
            for (int w = 0; w < VW / 4; ++w)
#pragma unroll
                for (int x = 0; x < 4; ++x) {
                    const bool bad = !finite(v.x[j][w][x]);
                    odd |= bad;
                    v.x[j][w][x] = bad ? 0.f : v.x[j][w][x];
                }
        return odd;
    }
    static constexpr bool TWO = false;
    struct P { f32x4 x[2]; };
    static __device__ __forceinline__ P probs(const f32x4 (&s)[2]) { return {s[0], s[1]}; }
    static __device__ __forceinline__ f32x4 pv(const V& v, int e, const P& p, f32x4 o) {
#pragma unroll
        for (int j = 0; j < 8; ++j) o = __builtin_amdgcn_mfma_f32_16x16x4f32(v.x[j][e >> 2][e & 3], p.x[j >> 2][j & 3], o, 0, 0, 0);
        return o;
    }
};

// max / sum over the four lanes that hold one row's keys (lanes i, i + 16, i + 32, i + 48)
__device__ __forceinline__ float max_over_groups(float v) {
    unsigned u = __builtin_bit_cast(unsigned, v);
    auto s = __builtin_amdgcn_permlane16_swap(u, u, false, false);
    v = fmaxf(__builtin_bit_cast(float, (unsigned)s[0]), __builtin_bit_cast(float, (unsigned)s[1]));
    u = __builtin_bit_cast(unsigned, v);
    s = __builtin_amdgcn_permlane32_swap(u, u, false, false);
    return fmaxf(__builtin_bit_cast(float, (unsigned)s[0]), __builtin_bit_cast(float, (unsigned)s[1]));
}

// The pages of tile kt (keys 32 kt ..): uniform over the wave.  An entry that names no page leaves its keys unseen.
struct TilePages { int p0, p1; };
__device__ __forceinline__ TilePages tile_pages(const AttnArgs& a, const int* row, int kt) {
    TilePages t;
    const int j = (kt * 32) >> a.shift;
    t.p0 = row[min(j, a.width - 1)];
    t.p1 = a.shift == 4 ? row[min(j + 1, a.width - 1)] : t.p0;
    return t;
}
template <typename F, typename T>
__device__ __forceinline__ void load_tile(const AttnArgs& a, typename F::K& k, typename F::V& v, TilePages t, int kt, int hk, int i, int g, int D) {
    const bool two = a.shift == 4;
    const long p0 = (unsigned)t.p0 < (unsigned)a.n_pages ? t.p0 : 0, p1 = (unsigned)t.p1 < (unsigned)a.n_pages ? t.p1 : 0;
    const long off = (long)((kt * 32) & ((1 << a.shift) - 1)) * D;
    const T* k0 = (const T*)a.k + p0 * a.sp + hk * a.sh + off;
    const T* k1 = (const T*)a.k + p1 * a.sp + hk * a.sh + off;
    const T* v0 = (const T*)a.v + p0 * a.svp + hk * a.svh + off;
    const T* v1 = (const T*)a.v + p1 * a.svp + hk * a.svh + off;
    F::load_k(k, k0, k1, two, i, g);
    F::load_v(v, v0, v1, two, i, g);
}

// Running softmax of NT tiles of 16 rows: m in the exponent's units (base 2), l each lane's own keys only.
template <int NT, int D> struct State {
    f32x4 o[NT][D / 16];
    float m[NT], l[NT];
    __device__ __forceinline__ void clear() {
#pragma unroll
        for (int n = 0; n < NT; ++n) {
            m[n] = -INFINITY; l[n] = 0.f;
#pragma unroll
            for (int e = 0; e < D / 16; ++e) o[n][e] = (f32x4){0.f, 0.f, 0.f, 0.f};
        }
    }
};

// One tile of 32 keys into the state.  limit[n]: the last key the lane's row of tile n sees; kmin / kmax: the smallest /
// largest of them over the wave's rows (a tile that ends at or before kmin needs no comparison).  In a tile that some row
// sees in part, values behind every row's last key are cleared, and ones that are not finite (0 * inf for a row that does
// not see them) are left out of the product and added to the rows that do.
template <typename F, int NT, int D>
__device__ __forceinline__ void attend_tile(State<NT, D>& st, const typename F::Q (&q)[NT], const typename F::K& k, typename F::V& v,
                                            const int (&limit)[NT], int hk, int kt, int kmin, int kmax, TilePages tp, const AttnArgs& a, int lane) {
    typedef typename F::T T;
    const int g = lane >> 4, k0 = kt * 32;
    const bool bad0 = (unsigned)tp.p0 >= (unsigned)a.n_pages, bad1 = (unsigned)tp.p1 >= (unsigned)a.n_pages;
    const bool whole = !bad0 && !bad1 && k0 + 31 <= kmin;
    bool odd = false;
    if (!whole) {
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const int key = F::key_of_v(j, g);
            if (k0 + key > kmax || ((key & 16) ? bad1 : bad0)) F::zero_key(v, j);
        }
        odd = __any(F::keep_finite(v));
    }
#pragma unroll
    for (int n = 0; n < NT; ++n) {
        f32x4 s[2];
        F::scores(s, k, q[n]);
#pragma unroll
        for (int t = 0; t < 2; ++t)
#pragma unroll
            for (int r = 0; r < 4; ++r) s[t][r] *= a.c;
        if (!whole) {
#pragma unroll
            for (int t = 0; t < 2; ++t)
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    const int key = F::key_of_score(t, r, g);
                    if (k0 + key > limit[n] || ((key & 16) ? bad1 : bad0)) s[t][r] = -INFINITY;
                }
        }
        float mx = fmaxf(fmaxf(fmaxf(s[0][0], s[0][1]), fmaxf(s[0][2], s[0][3])), fmaxf(fmaxf(s[1][0], s[1][1]), fmaxf(s[1][2], s[1][3])));
        mx = fmaxf(st.m[n], max_over_groups(mx));
        if (__any(mx > st.m[n])) {                     // some row's maximum moved
            const float al = mx == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(st.m[n] - mx);
            st.m[n] = mx;
            st.l[n] *= al;
#pragma unroll
            for (int e = 0; e < D / 16; ++e) st.o[n][e] *= al;
        }
        const float ref = mx == -INFINITY ? 0.f : mx;   // a row that has seen nothing yet: all its exponentials are 0
        float sum = 0.f;
#pragma unroll
        for (int t = 0; t < 2; ++t)
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                s[t][r] = __builtin_amdgcn_exp2f(s[t][r] - ref);
                sum += s[t][r];
            }
        st.l[n] += sum;
        const typename F::P p = F::probs(s);
#pragma unroll
        for (int e = 0; e < D / 16; ++e) st.o[n][e] = F::pv(v, e, p, st.o[n][e]);
    }
    if (odd) {
#pragma unroll 1
        for (int key = 0; key < 32; ++key) {
            if (k0 + key > kmax || ((key & 16) && a.shift == 4 ? bad1 : bad0)) continue;
            const long page = (key & 16) && a.shift == 4 ? tp.p1 : tp.p0;
            const T* p = (const T*)a.v + page * a.svp + hk * a.svh + (long)((k0 + key) & ((1 << a.shift) - 1)) * D + (D / 4) * g;
#pragma unroll
            for (int r = 0; r < 4; ++r)
#pragma unroll
                for (int e = 0; e < D / 16; ++e) {
                    const float f = to_f32<T>(p[(D / 16) * r + e]);
#pragma unroll
                    for (int n = 0; n < NT; ++n) st.o[n][e][r] += !finite(f) && k0 + key <= limit[n] ? f : 0.f;
                }
        }
    }
}

// Tiles first, first + step, ... < end of the request's keys.  AHEAD: the next tile's keys and values are in flight while a
// tile is computed, its page numbers one tile further ahead; without, other waves' tiles are.  `loaded`: tile `first` is
// already on its way.  An infinite value times a probability's second piece, which may be 0 or negative, is NaN where the first
// piece alone gives an infinity: if that happens the tiles are gone through again as ones that a row sees in part.  Nothing else changes by it.
template <typename F> struct Stage { typename F::K k; typename F::V v; TilePages tp; };
template <typename F, typename T, int NT, int D, bool AHEAD>
__device__ __forceinline__ void attend(State<NT, D>& st, const AttnArgs& a, const typename F::Q (&q)[NT], const int (&limit)[NT],
                                       const int* row, int hk, int first, int step, int end, int kmin, int kmax, int lane,
                                       Stage<F> (&sg)[AHEAD ? 2 : 1], bool loaded) {
    if (first >= end) return;
    const int i = lane & 15, g = lane >> 4;
    TilePages next;
    auto compute = [&](int kt, Stage<F>& s) {
        attend_tile<F, NT, D>(st, q, s.k, s.v, limit, hk, kt, kmin, kmax, s.tp, a, lane);
    };
    auto fetch = [&](int kt, Stage<F>& s) {
        s.tp = next;
        load_tile<F, T>(a, s.k, s.v, next, kt, hk, i, g, D);
        next = tile_pages(a, row, kt + step);
    };
    for (bool again = false;; again = true) {
        if (!loaded) {
            sg[0].tp = tile_pages(a, row, first);
            load_tile<F, T>(a, sg[0].k, sg[0].v, sg[0].tp, first, hk, i, g, D);
        }
        next = tile_pages(a, row, first + step);
        if constexpr (AHEAD) {
            for (int kt = first; kt < end; kt += 2 * step) {
                if (kt + step < end) fetch(kt + step, sg[1]);
                compute(kt, sg[0]);
                if (kt + step < end) {
                    if (kt + 2 * step < end) fetch(kt + 2 * step, sg[0]);
                    compute(kt + step, sg[1]);
                }
            }
        } else {
            for (int kt = first; kt < end; kt += step) {
                compute(kt, sg[0]);
                if (kt + step < end) fetch(kt + step, sg[0]);
            }
        }
        bool nan = false;
        if (F::TWO && !again) {
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
                for (int e = 0; e < D / 16; ++e)
#pragma unroll
                    for (int r = 0; r < 4; ++r) nan |= st.o[n][e][r] != st.o[n][e][r] && st.l[n] == st.l[n];
        }
        if (!__any(nan)) return;
        st.clear();
        loaded = false;
        kmin = -1;
    }
}

template <int D> __device__ __forceinline__ void store_vals(bf16_t* p, const float* x) {
#pragma unroll
    for (int c = 0; c < D / 32; ++c) {
        bf16x8 o;
#pragma unroll
        for (int j = 0; j < 8; ++j) o[j] = (bf16_t)x[8 * c + j];
        *(bf16x8*)(p + 8 * c) = o;
    }
}
template <int D> __device__ __forceinline__ void store_vals(float* p, const float* x) {
#pragma unroll
    for (int c = 0; c < D / 16; ++c) *(f32x4*)(p + 4 * c) = *(const f32x4*)(x + 4 * c);
}

// ---- few rows: the WAVES waves of a workgroup take the tiles of the keys in turn and are merged through LDS; a split
// grid leaves {m, l} and O of every row and split to paged_attn_join_kernel.  One row would do with vector instructions, but
// 16 cost the matrix pipe nothing that the memory would not take longer for, probabilities in two pieces included (one piece: the same
// times, 0.4 us less for the smallest): 64 requests x 20 heads x 1500 keys (492 MB) in 86 us, 5.7 TB/s, the rate of a long read;
// 4 requests of 7000 to 32700 keys, 8 heads of 128 (271 MB), 56 us and 5 for the join; 8 requests x 6 heads x 440 keys 7.5 us, a
// launch and three dependent trips to memory.
template <int D, int WAVES> struct FewLds { float m[WAVES][16], l[WAVES][16], o[WAVES][16][D + 4]; };
template <typename T, int D, int WAVES, bool AHEAD>
__device__ __forceinline__ void attn_few(const AttnArgs& a, FewLds<D, WAVES>& lds, int bx, int by, int ny) {
    typedef Frag<T, D> F;
    const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int i = lane & 15, g = lane >> 4;
    const int split = bx % a.splits, x = bx / a.splits;
    const int hk = x % a.Hk, b = x / a.Hk;
    const int* row = a.table + b * a.ld_table;
    Stage<F> sg[AHEAD ? 2 : 1];
    // the first tile does not depend on the request's length: it is under way while that is read
    bool loaded = AHEAD && a.splits == 1 && (w * 32) >> a.shift < a.width;
    if (loaded) {
        sg[0].tp = tile_pages(a, row, w);
        load_tile<F, T>(a, sg[0].k, sg[0].v, sg[0].tp, w, hk, i, g, D);
    }
    const Req r = request(a, b);
    const int rows = r.nq * a.G;
    if (a.few_rows && rows > a.few_rows) return;
    for (int r0 = by * 16; r0 < rows; r0 += ny * 16) {
        const int n_rows = min(16, rows - r0);
        const int tok0 = r0 / a.G, tok1 = (r0 + n_rows - 1) / a.G;
        const int base = a.causal ? r.len - r.nq : r.len - 1;               // last key of token t: base + t (causal) or base
        const int kmin = a.causal ? base + tok0 : base, kmax = a.causal ? base + tok1 : base;
        const int my = r0 + min(i, n_rows - 1), tok = my / a.G, head = hk * a.G + my - tok * a.G;
        typename F::Q q[1];
        F::load_q(q[0], (const T*)a.q + (long)(r.q0 + tok) * a.ldq + (long)head * a.hq, g, i < n_rows);
        const int limit[1] = {i < n_rows ? (a.causal ? base + tok : base) : -1};
        State<1, D> st;
        st.clear();
        const int tiles = kmax >= 0 ? (kmax >> 5) + 1 : 0;
        const int per = (tiles + a.splits - 1) / a.splits, t0 = split * per, t1 = min(tiles, t0 + per);
        attend<F, T, 1, D, AHEAD>(st, a, q, limit, row, hk, t0 + w, WAVES, t1, kmin, kmax, lane, sg, loaded);
        loaded = false;
        st.l[0] = xor_add<32>(xor_add<16>(st.l[0]));
        if (g == 0) { lds.m[w][i] = st.m[0]; lds.l[w][i] = st.l[0]; }
        if (i < n_rows) {
#pragma unroll
            for (int rr = 0; rr < 4; ++rr)
#pragma unroll
                for (int e = 0; e < D / 16; ++e) lds.o[w][i][(D / 4) * g + (D / 16) * rr + e] = st.o[0][e][rr];
        }
        __syncthreads();
        // 8 columns a thread
        for (int c = threadIdx.x; c < n_rows * (D / 8); c += 64 * WAVES) {
            const int rw = c / (D / 8), d = (c % (D / 8)) * 8;
            float m = lds.m[0][rw];
#pragma unroll
            for (int u = 1; u < WAVES; ++u) m = fmaxf(m, lds.m[u][rw]);
            const float ref = m == -INFINITY ? 0.f : m;
            float l = 0.f, o[8];
#pragma unroll
            for (int j = 0; j < 8; ++j) o[j] = 0.f;
#pragma unroll
            for (int u = 0; u < WAVES; ++u) {
                const float f = __builtin_amdgcn_exp2f(lds.m[u][rw] - ref);
                l = fmaf(f, lds.l[u][rw], l);
#pragma unroll
                for (int j = 0; j < 8; ++j) o[j] = fmaf(f, lds.o[u][rw][d + j], o[j]);
            }
            const int t = (r0 + rw) / a.G, h = hk * a.G + (r0 + rw) - t * a.G;
            if (a.splits == 1) {
                const float inv = l == 0.f ? 0.f : 1.f / l;
#pragma unroll
                for (int j = 0; j < 8; ++j) o[j] *= inv;
                store_vals<32>((T*)a.o + (long)(r.q0 + t) * a.ldo + (long)h * a.ho + d, o);
            } else {
                const long y = ((long)(r.q0 + t) * (a.Hk * a.G) + h) * a.splits + split;
                store_vals<32>(a.part + y * D + d, o);
                if (d == 0) *(f32x2*)(a.part_ml + y * 2) = (f32x2){m, l};
            }
        }
        __syncthreads();
    }
}
template <typename T, int D, int WAVES, bool AHEAD>
__global__ __launch_bounds__(64 * WAVES, D == 128 ? 2 : sizeof(T) == 4 || AHEAD ? 3 : 4) void paged_attn_few_kernel(AttnArgs a) {
    __shared__ FewLds<D, WAVES> lds;
    attn_few<T, D, WAVES, AHEAD>(a, lds, blockIdx.x, blockIdx.y, gridDim.y);
}

// Joins the splits of a row, a wave per row: lane s weighs split s, then every lane adds up its columns.
template <typename T, int D>
__global__ __launch_bounds__(256) void paged_attn_join_kernel(AttnArgs a) {
    const int lane = threadIdx.x & 63;
    const long H = (long)a.Hk * a.G, rows = H * a.N;
    const long x = (long)blockIdx.x * 4 + (threadIdx.x >> 6);
    if (x >= rows) return;
    const int t = (int)(x / H), h = (int)(x - t * H);
    if (t < a.q_start[0] || t >= a.q_start[a.B]) return;       // rows of no request were not written, and stay as they are
    const f32x2 ml = lane < a.splits ? *(const f32x2*)(a.part_ml + (x * a.splits + lane) * 2) : (f32x2){-INFINITY, 0.f};
    const float m = wave_max(ml[0]);
    float w = m == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(ml[0] - m);
    const float l = wave_sum(w * ml[1]);
    w *= l == 0.f ? 0.f : 1.f / l;
    const float* p = a.part + x * a.splits * D + lane * (D / 64);
    float o[D / 64];
#pragma unroll
    for (int c = 0; c < D / 64; ++c) o[c] = 0.f;
    auto add = [&](int s0, int n) {                             // n splits from s0 on
#pragma unroll
        for (int u = 0; u < n; ++u) {
            const float f = __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, w), s0 + u));
#pragma unroll
            for (int c = 0; c < D / 64; ++c) o[c] = fmaf(f, p[(long)(s0 + u) * D + c], o[c]);
        }
    };
    int s0 = 0;
    for (; s0 + 8 <= a.splits; s0 += 8) add(s0, 8);             // eight loads in flight
    if (a.splits & 4) { add(s0, 4); s0 += 4; }
    if (a.splits & 2) { add(s0, 2); s0 += 2; }
    if (a.splits & 1) add(s0, 1);
    T* out = (T*)a.o + (long)t * a.ldo + (long)h * a.ho + lane * (D / 64);
#pragma unroll
    for (int c = 0; c < D / 64; ++c) out[c] = from_f32<T>(o[c]);
}

// ---- many rows.  The row tiles of all requests (TR rows each) are dealt out with the longest request's first, so that the
// last workgroups to start are short ones: their work goes with the number of keys.  The order is found by every workgroup
// for itself, a lane per request; with more than 64 requests, tiles are numbered in the requests' order, request b's from
// q_start[b]*G/TR + b on (one more than it can fill, so that no sum is needed).
struct RowTile { Req r; int b, rows, r0; };
template <int TR> __device__ __forceinline__ RowTile row_tile(const AttnArgs& a, int tile, int lane) {
    RowTile t;
    int start;
    if (a.B <= 64) {
        Req r = {0, 0, 0};
        if (lane < a.B) r = request(a, lane);
        const int mine = r.nq * a.G > a.few_rows ? (r.nq * a.G + TR - 1) / TR : 0;
        int before = 0, total = 0;
        for (int j = 0; j < a.B; ++j) {
            const int len = __builtin_amdgcn_readlane(r.len, j), n = __builtin_amdgcn_readlane(mine, j);
            before += len > r.len || (len == r.len && j < lane) ? n : 0;
            total += n;
        }
        // the workgroups that start together on a CU: one of the longest, one of the shortest, one from between
        const int round = max(1, 256 / (a.Hk * a.splits));
        if (tile >= round && tile < total) tile = tile < 2 * round ? total - 1 - (tile - round) : tile - round;
        const unsigned long long who = __ballot(tile >= before && tile < before + mine);
        t.b = who ? __builtin_ctzll(who) : 0;
        start = who ? __builtin_amdgcn_readlane(before, t.b) : 1 << 30;      // no such tile
    } else {
        int lo = 0, hi = a.B;
        while (hi - lo > 1) {
            const int mid = (lo + hi) >> 1;
            if ((int)((long)a.q_start[mid] * a.G / TR) + mid <= tile) lo = mid; else hi = mid;
        }
        t.b = lo;
        start = (int)((long)a.q_start[lo] * a.G / TR) + lo;
    }
    t.r = request(a, t.b);
    t.rows = t.r.nq * a.G;
    t.r0 = start > tile ? -(1 << 30) : (tile - start) * TR;
    if (a.causal && t.r0 >= 0) t.r0 = ((t.rows + TR - 1) / TR - 1) * TR - t.r0;     // the last rows see the most
    return t;
}
// fp32: each of the four waves takes 16 NT rows of the tile and walks its keys, straight from the pages; bound by the fp32
// matrix instructions (4 requests of 512 tokens on 2048 keys, 8 heads: 124 us, 61 TF of the 150 that a large product reaches).
template <typename T, int D, int NT>
__global__ __launch_bounds__(256) void paged_attn_rows_kernel(AttnArgs a) {
    typedef Frag<T, D> F;
    const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int i = lane & 15, g = lane >> 4;
    const int hk = blockIdx.x % a.Hk, split = blockIdx.x / a.Hk % a.splits, tile = blockIdx.x / a.Hk / a.splits;
    const RowTile rt = row_tile<64 * NT>(a, tile, lane);
    const Req r = rt.r;
    const int rows = rt.rows, r0 = rt.r0 + w * 16 * NT;
    if (rows <= a.few_rows || r0 < 0 || r0 >= rows) return;
    const int n_rows = min(16 * NT, rows - r0);
    const int base = a.causal ? r.len - r.nq : r.len - 1;
    const int kmin = a.causal ? base + r0 / a.G : base, kmax = a.causal ? base + (r0 + n_rows - 1) / a.G : base;
    typename F::Q q[NT];
    int limit[NT];
#pragma unroll
    for (int n = 0; n < NT; ++n) {
        const bool ok = 16 * n + i < n_rows;
        const int my = r0 + (ok ? 16 * n + i : 0), tok = my / a.G, head = hk * a.G + my - tok * a.G;
        F::load_q(q[n], (const T*)a.q + (long)(r.q0 + tok) * a.ldq + (long)head * a.hq, g, ok);
        limit[n] = ok ? (a.causal ? base + tok : base) : -1;
    }
    State<NT, D> st;
    st.clear();
    const int tiles = kmax >= 0 ? (kmax >> 5) + 1 : 0, per = (tiles + a.splits - 1) / a.splits, t0 = split * per;
    Stage<F> sg[2];
    attend<F, T, NT, D, true>(st, a, q, limit, a.table + rt.b * a.ld_table, hk, t0, 1, min(tiles, t0 + per), kmin, kmax, lane, sg, false);
#pragma unroll
    for (int n = 0; n < NT; ++n) {
        const float l = xor_add<32>(xor_add<16>(st.l[n]));
        const float inv = a.splits > 1 ? 1.f : l == 0.f ? 0.f : 1.f / l;
        if (16 * n + i >= n_rows) continue;
        const int my = r0 + 16 * n + i, tok = my / a.G, head = hk * a.G + my - tok * a.G;
        float o[D / 4];
#pragma unroll
        for (int rr = 0; rr < 4; ++rr)
#pragma unroll
            for (int e = 0; e < D / 16; ++e) o[(D / 16) * rr + e] = st.o[n][e][rr] * inv;
        if (a.splits == 1) store_vals<D>((T*)a.o + (long)(r.q0 + tok) * a.ldo + (long)head * a.ho + (D / 4) * g, o);
        else {
            const long x = ((long)(r.q0 + tok) * (a.Hk * a.G) + head) * a.splits + split;
            store_vals<D>(a.part + x * D + (D / 4) * g, o);
            if (g == 0) *(f32x2*)(a.part_ml + x * 2) = (f32x2){st.m[n], l};
        }
    }
}

// bf16: tiles of 64 keys go to LDS once for the workgroup's four waves of 32 rows (LDS-DMA, two buffers, one barrier per
// tile).  S^T and O^T as above on v_mfma_f32_32x32x16_bf16 (A row / B column lane & 31, k = 8 (lane / 32) + j; C column
// lane & 31, row (i & 3) + 8 (i >> 2) + 4 (lane / 32)); V fragments come transposed out of LDS.  Per score the vector unit
// has a maximum, a multiply-add, an exponential, an addition, a subtraction and a conversion to do, more cycles than the matrix
// pipe needs for the products of a 64-column head: the maximum is only compared (the reference point moves when a score
// exceeds it by 2^8), the scale's sign is taken into Q so that raw scores can be compared.  16 requests of 512 tokens on
// 4096 keys, 16 heads over 4: 241 us (535 TF) with 64 columns, 200 us (645 TF) with 8 heads of 128.  With probabilities of one bf16
// value, two products of three, 169 and 148 us.
// Requests with few rows, bound by memory, are in the same grid: beside the matrix products of the others (64 requests of 1 to 512
// tokens on 1000 to 4000 keys, 16 heads over 4: 82 us, as two launches 119; 32 of 1 to 1000 on up to 6000, 32 heads of 128 over
// 8: 209, 266).  They start behind as many of the large ones as fill half the chip's places, which then lie evenly on the CUs: in
// front of all of them 64 requests of 1 to 224 tokens take 40 us, behind them 32 but the batch of 32 261, here 29 and 209.
__device__ __forceinline__ float max3(float a, float b, float c) {
    float r;
    asm("v_max3_f32 %0, %1, %2, %3" : "=v"(r) : "v"(a), "v"(b), "v"(c));
    return r;
}
// The compiler puts no wait between a matrix instruction and inline assembly that reads its result: scores pass through here
// before the maximum is taken of them straight away (12 wait states, what the compiler leaves before an instruction of its own).
__device__ __forceinline__ void settle(f32x16& a, f32x16& b) { asm volatile("s_nop 11" : "+v"(a), "+v"(b)); }
__device__ __forceinline__ float max16(const f32x16& s) {
    float a = max3(s[0], s[1], s[2]), b = max3(s[3], s[4], s[5]);
    a = max3(a, s[6], s[7]); b = max3(b, s[8], s[9]);
    a = max3(a, s[10], s[11]); b = max3(b, s[12], s[13]);
    return max3(max3(a, s[14], s[15]), b, b);
}
template <int D> struct KvTile {
    static constexpr int CH = D / 8;                                  // 16-byte chunks of a key row
    static constexpr int PIECES = 16 * CH / 64;                       // DMA instructions of 16 keys
    // chunk c of a row stands at c ^ swizzle(row), so that neither fragment read below hits a bank twice
    static __device__ __forceinline__ int kswz(int row) { return D == 64 ? (row >> 1) & 7 : row & 15; }
    static __device__ __forceinline__ int vswz(int row) { return D == 64 ? ((row >> 1) & 1) << 2 : (row & 3) << 2; }
    // A fragment is read at a lane's offset (bytes, the same for every run of 32 keys) plus a constant; the swizzle turns the column
    // into an exclusive or of it.  It is made anew for every read: kept, the offsets would take registers that the accumulators need.
    static __device__ __forceinline__ int flip(int off, int bits) {
        asm("" : "+v"(off));
        return off ^ bits;
    }
    // Keys: row lane & 31, columns 16 ks + 8 (lane / 32) ..
    static __device__ __forceinline__ int koff(int lane) {
        const int row = lane & 31;
        return (row * D + (((lane >> 5) ^ kswz(row)) << 3)) * 2;
    }
    static __device__ __forceinline__ bf16x8 kfrag(const char* K, int off, int ks) { return *(const bf16x8*)(K + (ks ? flip(off, 32 * ks) : off)); }
    // Values, transposed: columns 32 db + (lane & 31) of the keys 16 s2 + {0..3, 8..11} + 4 (lane / 32), the order of a score register's
    // keys.  16 lanes read four 32-byte pieces of four rows; which is a swizzle's bits do not depend on s2.
    static __device__ __forceinline__ int voff(int lane) {
        const int i16 = lane & 15, row = 4 * (lane >> 5) + (i16 >> 2), col = 16 * ((lane >> 4) & 1) + 4 * (i16 & 3);
        return (row * D + (((col >> 3) ^ vswz(row)) << 3) + (col & 7)) * 2;
    }
    static __device__ __forceinline__ bf16x8 vfrag(const char* V, int s2, int off, int db) {
        bf16x8 f;
        if (db) off = flip(off, 64 * db);
#pragma unroll
        for (int jh = 0; jh < 2; ++jh) {
            const char* p = V + off + (16 * s2 + 8 * jh) * D * 2;
            const bf16x4 t = __builtin_bit_cast(bf16x4, __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4*)p));
#pragma unroll
            for (int x = 0; x < 4; ++x) f[4 * jh + x] = t[x];
        }
        return f;
    }
};

// keys of half a dword each behind `last` cleared out of a V fragment (keys k0 + 16 s2 + ...)
__device__ __forceinline__ u32x4 cut_keys(u32x4 v, int first, int hf, int last) {
#pragma unroll
    for (int x = 0; x < 4; ++x) {
        const int key = first + 8 * (x >> 1) + 4 * hf + 2 * (x & 1);
        v[x] &= (key <= last ? 0xFFFFu : 0u) | (key + 1 <= last ? 0xFFFF0000u : 0u);
    }
    return v;
}
__device__ __forceinline__ u32x4 finite_part(u32x4 v, bool& odd) {
#pragma unroll
    for (int x = 0; x < 4; ++x) v[x] = finite_half(v[x], odd);
    return v;
}

template <int D>
__global__ __launch_bounds__(256, D == 64 ? 4 : 2) void paged_attn_chunk_kernel(AttnArgs a) {
    typedef KvTile<D> L;
    typedef bf16_t T;
    __shared__ union { struct { bf16_t k[2][64 * D], v[2][64 * D]; } kv; FewLds<D, 4> few; } lds __attribute__((aligned(16)));
    auto &Ks = lds.kv.k, &Vs = lds.kv.v;
    __shared__ int again;
    // The grid is runs of eight workgroups, one for each XCD, so that those of a kv head stay on theirs; the runs of requests with
    // few rows stand behind the first FIRST of the others.
    constexpr unsigned FIRST = D == 64 ? 64 : 32;
    const unsigned run = blockIdx.x >> 3, few_runs = (unsigned)(a.n_few + 7) >> 3, first_runs = min((gridDim.x >> 3) - few_runs, FIRST);
    if (run >= first_runs && run < first_runs + few_runs) {
        const int ny = a.few_tiles, nx = a.n_few / ny, at = (int)(blockIdx.x - 8 * first_runs);
        if (at < a.n_few) attn_few<T, D, 4, false>(a, lds.few, at % nx, at / nx, ny);
        return;
    }
    const int id = (int)(run < first_runs ? blockIdx.x : blockIdx.x - 8 * few_runs);
    const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int r32 = lane & 31, hf = lane >> 5;
    const int hk = id % a.Hk, split = id / a.Hk % a.splits, tile = id / a.Hk / a.splits;
    const RowTile rt = row_tile<128>(a, tile, lane);
    const Req r = rt.r;
    if (rt.rows <= a.few_rows || rt.r0 < 0 || rt.r0 >= rt.rows) return;
    const int wg_rows = min(128, rt.rows - rt.r0);
    const int base = a.causal ? r.len - r.nq : r.len - 1;
    const int kmin = a.causal ? base + rt.r0 / a.G : base;                           // the last key that all rows of the workgroup see
    const int kmax_wg = a.causal ? base + (rt.r0 + wg_rows - 1) / a.G : base;        // ... and that any of them sees
    // this wave's 32 rows; a wave without any helps to move the tiles
    const int r0 = rt.r0 + w * 32, n_rows = max(0, min(32, rt.rows - r0));
    const int kmax = n_rows == 0 ? -1 : a.causal ? base + (r0 + n_rows - 1) / a.G : base;
    const bool mine = r32 < n_rows;
    const int my = mine ? r0 + r32 : 0, tok = my / a.G, head = hk * a.G + my - tok * a.G;
    const int limit = mine ? (a.causal ? base + tok : base) : -1;
    bf16x8 q[D / 16];
    {
        const T* p = (const T*)a.q + (long)(r.q0 + tok) * a.ldq + (long)head * a.hq + 8 * hf;
        const unsigned flip = a.c < 0.f ? 0x80008000u : 0u;
#pragma unroll
        for (int ks = 0; ks < D / 16; ++ks) {
            u32x4 v = {0u, 0u, 0u, 0u};
            if (mine) v = *(const u32x4*)(p + 16 * ks);
#pragma unroll
            for (int x = 0; x < 4; ++x) v[x] ^= flip;
            q[ks] = __builtin_bit_cast(bf16x8, v);
        }
    }
    const float c = fmaxf(fabsf(a.c), 1e-37f);                    // never 0: -inf times it stays -inf
    const float lazy = 8.f / c;
    f32x16 o[D / 32];
#pragma unroll
    for (int d = 0; d < D / 32; ++d)
#pragma unroll
        for (int x = 0; x < 16; ++x) o[d][x] = 0.f;
    float m = -INFINITY, nm = 0.f, thr = -INFINITY, l = 0.f;      // reference point, -c times it, what moves it, row sum (this lane's keys)
    const int tiles = kmax_wg >= 0 ? (kmax_wg >> 6) + 1 : 0, per = (tiles + a.splits - 1) / a.splits;
    const int t0 = split * per, t1 = min(tiles, t0 + per);
    const int* row = a.table + rt.b * a.ld_table;
    // 64 entries of the block table, a lane each, from entry `first` on: a scalar would have to be fetched anew for every
    // tile behind the DMA's back, and its wait would be one for the DMA
    int first = t0 * 64 >> a.shift;
    int entries = t0 < t1 ? row[min(first + lane, a.width - 1)] : 0;
    // where the lane's 16 bytes of a DMA piece (64 / CH rows, 1 KiB) come from; piece u of a run: 1024 u further, a key's chunk at ^ 4 u
    const int lr = lane / L::CH, ch = lane & (L::CH - 1);
    const unsigned kmove = (lr * D + ((ch ^ L::kswz(lr)) << 3)) * 2, vmove = (lr * D + ((ch ^ L::vswz(lr)) << 3)) * 2;
    const int kr = L::koff(lane), vr = L::voff(lane);
    // Tile kt into a buffer; wave w moves run w of its four runs of 16 keys, of the keys and of the values.  Returns which of
    // the runs' pages exist.
    auto move = [&](int kt, int buf) {
        if (((kt * 64 + 48) >> a.shift) - first >= 64) {
            first = kt * 64 >> a.shift;
            entries = row[min(first + lane, a.width - 1)];
            asm volatile("" : "+v"(entries));                     // its wait belongs in here: outside it would drain the DMA every time
        }
        unsigned have = 0;
#pragma unroll
        for (int u = 0; u < 4; ++u)
            have |= ((unsigned)__builtin_amdgcn_readlane(entries, ((kt * 64 + 16 * u) >> a.shift) - first) < (unsigned)a.n_pages ? 1u : 0u) << u;
        const int pw = __builtin_amdgcn_readlane(entries, ((kt * 64 + 16 * w) >> a.shift) - first);
        const long page = (unsigned)pw < (unsigned)a.n_pages ? pw : 0;
        const int in = (kt * 64 + 16 * w) & ((1 << a.shift) - 1);
        const char* k = (const char*)((const T*)a.k + page * a.sp + hk * a.sh + in * D);
        const char* v = (const char*)((const T*)a.v + page * a.svp + hk * a.svh + in * D);
#pragma unroll
        for (int u = 0; u < L::PIECES; ++u) {
            dma_piece(k + 1024 * u, kmove ^ 64 * u, (const char*)&Ks[buf][(16 * w) * D + u * 512]);
            dma_piece(v + 1024 * u, vmove, (const char*)&Vs[buf][(16 * w) * D + u * 512]);
        }
        return have;
    };
    if (threadIdx.x == 0) again = 0;                             // set behind the barrier of the first tile at the earliest
    int kt = t0, buf = 0;
    unsigned next = t0 < t1 ? move(t0, 0) : 0;
    // Tile kt is in LDS for every wave, the next one on its way into the other buffer; which runs of this one have pages.
    auto arrive = [&]() {
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        __syncthreads();
        const unsigned have = next;
        if (kt + 1 < t1) next = move(kt + 1, buf ^ 1);
        return have;
    };
    // the reference point moves to the row's maximum so far (rare after the first tiles)
    auto move_reference = [&](float mx) {
        const unsigned u = __builtin_bit_cast(unsigned, mx);
        const auto sw = __builtin_amdgcn_permlane32_swap(u, u, false, false);
        const float top = fmaxf(m, fmaxf(__builtin_bit_cast(float, (unsigned)sw[0]), __builtin_bit_cast(float, (unsigned)sw[1])));
        const float al = top > m ? __builtin_amdgcn_exp2f((m - top) * c) : 1.f;
        m = top;
        thr = top + lazy;
        nm = top == -INFINITY ? 0.f : -(top * c);
        l *= al;
#pragma unroll
        for (int d = 0; d < D / 32; ++d)
#pragma unroll
            for (int x = 0; x < 16; ++x) o[d][x] *= al;
    };
    // Scores to probabilities, in two pieces for the product; the sum is of the whole ones.
    auto exponentials = [&](f32x16& s, bf16x8 (&hi)[2], bf16x8 (&lo)[2]) {
        float s0 = 0.f, s1 = 0.f;
#pragma unroll
        for (int x = 0; x < 16; x += 2) {
            s[x] = __builtin_amdgcn_exp2f(fmaf(s[x], c, nm));
            s[x + 1] = __builtin_amdgcn_exp2f(fmaf(s[x + 1], c, nm));
            s0 += s[x];
            s1 += s[x + 1];
        }
        l += s0 + s1;
#pragma unroll
        for (int x = 0; x < 16; x += 2) {
            const Two t = two_pieces(s[x], s[x + 1]);
            hi[x >> 3][x & 7] = t.hi[0]; hi[x >> 3][(x & 7) + 1] = t.hi[1];
            lo[x >> 3][x & 7] = t.lo[0]; lo[x >> 3][(x & 7) + 1] = t.lo[1];
        }
    };
    auto product = [&](bf16x8 v, bf16x8 hi, bf16x8 lo, f32x16& o) {
        o = __builtin_amdgcn_mfma_f32_32x32x16_bf16(v, lo, o, 0, 0, 0);
        o = __builtin_amdgcn_mfma_f32_32x32x16_bf16(v, hi, o, 0, 0, 0);
    };
    auto scores = [&](const char* K, f32x16& s) {
#pragma unroll
        for (int x = 0; x < 16; ++x) s[x] = 0.f;
#pragma unroll
        for (int ks = 0; ks < D / 16; ++ks) s = __builtin_amdgcn_mfma_f32_32x32x16_bf16(L::kfrag(K, kr, ks), q[ks], s, 0, 0, 0);
    };
    // A tile that every row sees whole, 64 keys at once: one look at the maximum, and the matrix pipe has the other half's
    // products to do while the vector unit makes the exponentials of one.
    auto whole_tile = [&]() {
        const char *K = (const char*)Ks[buf], *V = (const char*)Vs[buf];
        f32x16 s[2];
        scores(K, s[0]);
        scores(K + 64 * D, s[1]);
        settle(s[0], s[1]);
        const float mx = fmaxf(max16(s[0]), max16(s[1]));
        if (__any(mx > thr)) move_reference(mx);
#pragma unroll
        for (int st = 0; st < 2; ++st) {
            bf16x8 hi[2], lo[2];
            exponentials(s[st], hi, lo);
#pragma unroll
            for (int s2 = 0; s2 < 2; ++s2)
#pragma unroll
                for (int d = 0; d < D / 32; ++d) product(L::vfrag(V + st * 64 * D, s2, vr, d), hi[s2], lo[s2], o[d]);
        }
    };
    // 32 keys of a tile that some row sees in part: values behind every row's last key are cleared, and ones that are not finite
    // (0 * inf for a row that does not see them) are left out of the product and added to the rows that do.
    auto half_tile = [&](int st, unsigned have) {
        const char *K = (const char*)Ks[buf] + st * 64 * D, *V = (const char*)Vs[buf] + st * 64 * D;
        const int k0 = kt * 64 + 32 * st;
        const bool ok0 = have >> (2 * st) & 1, ok1 = have >> (2 * st + 1) & 1;
        f32x16 s;
        scores(K, s);
#pragma unroll
        for (int x = 0; x < 16; ++x) {
            const int key = (x & 3) + 8 * (x >> 2) + 4 * hf;
            if (k0 + key > limit || !(x < 8 ? ok0 : ok1)) s[x] = -INFINITY;
        }
        const float mx = max16(s);
        if (__any(mx > thr)) move_reference(mx);
        bf16x8 hi[2], lo[2];
        exponentials(s, hi, lo);
        bool odd = false;
#pragma unroll
        for (int s2 = 0; s2 < 2; ++s2)
#pragma unroll
            for (int d = 0; d < D / 32; ++d) {
                const u32x4 vf = cut_keys(__builtin_bit_cast(u32x4, L::vfrag(V, s2, vr, d)), k0 + 16 * s2, hf, (s2 ? ok1 : ok0) ? kmax : -1);
                product(__builtin_bit_cast(bf16x8, finite_part(vf, odd)), hi[s2], lo[s2], o[d]);
            }
        if (__any(odd)) {
#pragma unroll 1
            for (int key = 0; key < 32; ++key)
#pragma unroll
                for (int d = 0; d < D / 32; ++d)
#pragma unroll
                    for (int y = 0; y < 4; ++y) {
                        const int col = 32 * d + 8 * y + 4 * hf;
                        const bf16x4 v = *(const bf16x4*)(V + (key * D + (((col >> 3) ^ L::vswz(key)) << 3) + (col & 7)) * 2);
#pragma unroll
                        for (int z = 0; z < 4; ++z) {
                            const float f = (float)v[z];
                            o[d][4 * y + z] += !finite(f) && k0 + key <= limit && (key < 16 ? ok0 : ok1) ? f : 0.f;
                        }
                    }
        }
    };
    // two loops: with one, the accumulators would be copied where its two branches meet, for every tile
    unsigned have = 15u;
    for (; kt < t1 && kt * 64 + 63 <= kmin; ++kt, buf ^= 1) {
        have = arrive();
        if (have != 15u) break;
        whole_tile();
    }
    if (kt > t0) {
        // An infinite value times a probability's second piece, which may be 0 or negative, is NaN where the first piece alone gives an
        // infinity.  Every row sees these tiles whole: if it happened in one, the workgroup goes through them again by the second loop.
        bool nan = false;
#pragma unroll
        for (int d = 0; d < D / 32; ++d)
#pragma unroll
            for (int x = 0; x < 16; ++x) nan |= o[d][x] != o[d][x] && l == l;
        if (__any(nan)) again = 1;
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");         // the tile under way too: its buffer may be filled anew
        __syncthreads();
        if (again) {
#pragma unroll
            for (int d = 0; d < D / 32; ++d)
#pragma unroll
                for (int x = 0; x < 16; ++x) o[d][x] = 0.f;
            m = thr = -INFINITY;
            nm = l = 0.f;
            kt = t0;
            buf = 0;
            have = 15u;
            first = t0 * 64 >> a.shift;
            entries = row[min(first + lane, a.width - 1)];
            next = move(t0, 0);
        }
    }
    for (bool here = have != 15u; kt < t1; ++kt, buf ^= 1, here = false) {
        if (!here) have = arrive();
        if (kt * 64 > kmax) continue;                             // none of this wave's rows sees the tile
#pragma unroll 1
        for (int st = 0; st < 2; ++st) half_tile(st, have);
    }
    const float sum = xor_add<32>(l);
    if (!mine) return;
    const float inv = a.splits > 1 ? 1.f : sum == 0.f ? 0.f : 1.f / sum;
    const long x = ((long)(r.q0 + tok) * (a.Hk * a.G) + head) * a.splits + split;
    T* out = (T*)a.o + (long)(r.q0 + tok) * a.ldo + (long)head * a.ho;
#pragma unroll
    for (int d = 0; d < D / 32; ++d)
#pragma unroll
        for (int y = 0; y < 4; ++y) {
            f32x4 v;
            bf16x4 b;
#pragma unroll
            for (int z = 0; z < 4; ++z) { v[z] = o[d][4 * y + z] * inv; b[z] = (bf16_t)v[z]; }
            if (a.splits == 1) *(bf16x4*)(out + 32 * d + 8 * y + 4 * hf) = b;
            else *(f32x4*)(a.part + x * D + 32 * d + 8 * y + 4 * hf) = v;
        }
    if (a.splits > 1 && hf == 0) *(f32x2*)(a.part_ml + x * 2) = (f32x2){m * c, sum};
}

// Requests of up to FEW_ROWS rows (tokens times the heads that share a kv head) go to the first kernel: 16 requests of 500 to
// 4000 keys, 64 rows each, 26.9 us there and 27.8 in the second, 128 rows 45.9 and 32.1.
#define FEW_ROWS 64
struct AttnPlan { bool ahead; int waves, splits, tiles_few, few_rows, chunk_rows; bool few, chunk; int64_t chunk_tiles, grid_few, grid_chunk, floats; };
static AttnPlan attn_plan(int dtype, int64_t D, int64_t N, int64_t B, int64_t Hk, int64_t G, int64_t max_q, int64_t max_k) {
    AttnPlan p;
    if (max_q > N) max_q = N;                                  // here, so that the size query and the call make one plan of one bound
    const int64_t rows = max_q * G;
    p.chunk = rows > FEW_ROWS;
    p.few = !(p.chunk && B == 1 && N * G > FEW_ROWS);          // one large request: nothing for the first kernel
    p.few_rows = p.few && p.chunk ? FEW_ROWS : 0;
    p.tiles_few = (int)((rows < FEW_ROWS ? rows : FEW_ROWS) + 15) / 16;
    p.chunk_rows = dtype == AVSR_F32 ? (D == 64 ? 128 : 64) : 128;
    p.chunk_tiles = p.chunk ? N * G / p.chunk_rows + B : 0;
    // Key splits where the row tiles do not fill the chip (256 CUs).  The first kernel is given up to 768 workgroups of four
    // waves (three fit on a CU; where a key takes more than 128 bytes, two fit, and twice as many even out ragged lengths:
    // 32 requests of 1000 to 8000 keys, 8 heads of 128, 107 -> 95 us), of 128 keys at least; up to 512 keys are not split, the
    // join would cost more (3 us of 10).  The second kernel: up to 512 workgroups of 256 keys at least.
    const int64_t wgs = p.chunk ? Hk * p.chunk_tiles : B * Hk * p.tiles_few, bytes = D * (dtype == AVSR_F32 ? 4 : 2);
    const int64_t fill = (p.chunk ? 512 : bytes <= 128 ? 768 : 1536) / wgs, most = p.chunk ? (max_k + 255) / 256 : max_k <= 512 ? 1 : (max_k + 127) / 128;
    const int64_t s = fill < most ? fill : most;
    p.splits = (int)(s < 1 ? 1 : s > 64 ? 64 : s);
    // Eight waves where the workgroups leave CUs free.  The next tile ahead of time where a wave has a long way to go (64
    // requests x 20 heads of 1500 keys 92 -> 86 us) or all workgroups run at once anyway (40 requests x 8 heads of 60 to 448 keys
    // 11.2 -> 10.4 us); with more and short ones, more waves are better (64 x 20 of 20 to 440 keys 15.1 us, 17 ahead).  Only 128
    // bytes a key leave registers for it.
    const int64_t rows_tiles = B * p.tiles_few < N * G / 16 + B ? B * p.tiles_few : N * G / 16 + B;
    p.waves = p.few && wgs * p.splits <= 256 ? 8 : 4;
    p.ahead = bytes <= 128 && (p.waves == 8 || max_k > 512 || rows_tiles * Hk * p.splits <= 768);
    p.grid_few = p.few ? B * Hk * p.splits : 0;
    p.grid_chunk = Hk * p.chunk_tiles * p.splits;
    p.floats = p.splits > 1 ? N * Hk * G * p.splits * (D + 2) : 0;
    return p;
}
extern "C" int64_t avsr_paged_attn_workspace_bytes(int dtype, int64_t N, int64_t B, int64_t Hq, int64_t Hk, int64_t head_dim, int64_t max_q,
                                                   int64_t max_k) {
    if (N <= 0 || B <= 0 || Hk <= 0 || Hq % Hk || max_q <= 0 || max_k <= 0) return 0;
    return attn_plan(dtype, head_dim, N, B, Hk, Hq / Hk, max_q, max_k).floats * 4;
}

template <typename T, int D>
static int launch_attn(hipStream_t s, AttnArgs a, const AttnPlan& p) {
    const dim3 few((unsigned)p.grid_few, p.tiles_few);
    constexpr bool small = sizeof(T) * D <= 128;
    if constexpr (sizeof(T) == 2) {
        if (p.chunk) hipLaunchKernelGGL((paged_attn_chunk_kernel<D>), dim3((unsigned)((p.grid_chunk + 7) / 8 + (a.n_few + 7) / 8) * 8), dim3(256), 0, s, a);
    }
    const bool first = p.few && !(sizeof(T) == 2 && p.chunk);
#define L(WAVES, AHEAD) hipLaunchKernelGGL((paged_attn_few_kernel<T, D, WAVES, AHEAD>), few, dim3(64 * WAVES), 0, s, a)
    if (first && p.waves == 8) L(8, small);
    else if (first && small && p.ahead) L(4, small);
    else if (first) L(4, false);
#undef L
    if constexpr (sizeof(T) == 4) {
        if (p.chunk) hipLaunchKernelGGL((paged_attn_rows_kernel<T, D, D == 64 ? 2 : 1>), dim3((unsigned)p.grid_chunk), dim3(256), 0, s, a);
    }
    if (p.splits > 1) hipLaunchKernelGGL((paged_attn_join_kernel<T, D>), dim3((unsigned)(((int64_t)a.N * a.Hk * a.G + 3) / 4)), dim3(256), 0, s, a);
    return avsr_launch_status();
}

extern "C" int avsr_paged_attn(avsr_stream_t stream, int dtype, const void* q, int64_t ldq, int64_t q_head, const void* k_pages,
                               int64_t k_page_stride, int64_t k_head_stride, const void* v_pages, int64_t v_page_stride,
                               int64_t v_head_stride, const int32_t* table, int64_t ld_table, int64_t width, const int32_t* lens,
                               const int32_t* q_start, void* o, int64_t ldo, int64_t o_head, int64_t N, int64_t B, int64_t Hq,
                               int64_t Hk, int64_t head_dim, int64_t page, int64_t n_pages, int64_t max_q, int64_t max_k,
                               float scale, int causal, void* workspace, int64_t workspace_bytes) {
    if (!q || !k_pages || !v_pages || !table || !lens || !q_start || !o) return AVSR_EINVAL;
    if (N < 0 || B <= 0 || Hk <= 0 || Hq <= 0 || Hq % Hk || width <= 0 || ld_table < width || n_pages <= 0 || max_q <= 0 || max_k <= 0) return AVSR_EINVAL;
    if (dtype != AVSR_F32 && dtype != AVSR_BF16) return AVSR_EINVAL;
    if (!(fabsf(scale * LOG2E) < INFINITY)) return AVSR_EINVAL;
    const int shift = page_shift(page);
    if (shift < 0 || (head_dim != 64 && head_dim != 128) || n_pages > (1LL << (30 - shift)) || width > (1LL << (30 - shift))) return AVSR_EUNSUPPORTED;
    const int64_t qm = dtype == AVSR_F32 ? 4 : 8;
    if (N <= 1) ldq = ldo = 0;                                  // the stride of a dimension of one is never used
    if (Hq == 1) q_head = o_head = 0;
    if (Hk == 1) k_head_stride = v_head_stride = 0;
    if (n_pages == 1) k_page_stride = v_page_stride = 0;
    if ((ldq | q_head | k_page_stride | k_head_stride | v_page_stride | v_head_stride | ldo | o_head) % qm ||
        ((uintptr_t)q | (uintptr_t)k_pages | (uintptr_t)v_pages | (uintptr_t)o) % 16) return AVSR_EUNSUPPORTED;
    if (N > (1 << 28) || N * Hq > (1LL << 30) || B > (1 << 24) || B * Hk > (1LL << 24)) return AVSR_EUNSUPPORTED;
    if (N == 0) return AVSR_OK;
    const int64_t mk = max_k < width * page ? max_k : width * page;       // fewer keys are never split more
    const AttnPlan p = attn_plan(dtype, head_dim, N, B, Hk, Hq / Hk, max_q, mk);
    if (p.floats && (!workspace || workspace_bytes < p.floats * 4 || (uintptr_t)workspace % 16)) return AVSR_EINVAL;
    const int64_t n_few = p.chunk ? p.grid_few * p.tiles_few : 0;
    // a launch has fewer than 2^32 threads
    if (p.grid_few > 0xffffff || p.grid_chunk + n_few > 0xfffff0 || (p.splits > 1 && N * Hq > 0x3ffffff)) return AVSR_EUNSUPPORTED;
    float* part = (float*)workspace;
    AttnArgs a = {q, ldq, q_head, k_pages, v_pages, k_page_stride, k_head_stride, v_page_stride, v_head_stride, table, ld_table, (int)width,
                  lens, q_start, o, ldo, o_head, (int)B, (int)Hk, (int)(Hq / Hk), (int)N, shift, (int)n_pages, scale * LOG2E, causal != 0,
                  p.splits, p.few_rows, (int)n_few, p.tiles_few, part, part ? part + N * Hq * p.splits * head_dim : nullptr};
    hipStream_t s = (hipStream_t)stream;
    if (dtype == AVSR_BF16) return head_dim == 64 ? launch_attn<bf16_t, 64>(s, a, p) : launch_attn<bf16_t, 128>(s, a, p);
    return head_dim == 64 ? launch_attn<float, 64>(s, a, p) : launch_attn<float, 128>(s, a, p);
}
