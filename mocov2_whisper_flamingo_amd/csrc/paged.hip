// Serving a decoder from a paged key / value cache.
//
//  * paged_plan_*: block tables, slot map and positions of one step from the requests' lengths, on the GPU.
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
// new tokens are rows start_b .. of the step.  The sums are a dependency of all output, so ONE workgroup makes them
// (1024 requests per pass); what follows is independent per token and page.  Up to PLAN_ONE tokens the same workgroup
// writes it (one launch: latency is all there is), above that a second launch spreads it over the chip.
#define PLAN_THREADS 1024
#define PLAN_ONE 8192

struct PlanArgs {
    const int* lens; const int* add; int* table; long ld_table; int width; int* ring; int n_pages; const int* pool;
    int* lens_out; int* pool_out; int B; int shift; int max_tokens; int* q_start; int* slots; int* positions; int* status;
    int* ws;                       // two-launch form: [3][B] old length, first page taken, first page given; [4] totals
};

__device__ __forceinline__ int wave_scan_incl(int v, int lane) {
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
        const int u = __shfl_up(v, o);
        if (lane >= o) v += u;
    }
    return v;
}

// what request b asks for; bad: what cannot be
__device__ __forceinline__ void plan_request(const PlanArgs& a, int b, int& len, int& need, int& give, int& more, int& bad) {
    len = need = give = more = 0;
    if (b >= a.B) return;
    len = a.lens[b];
    const int add = a.add[b];
    const long room = (long)a.width << a.shift;
    if (len < 0) { bad |= 8; len = 0; return; }
    if (len > room) { bad |= 2; return; }
    const int have = (len + (1 << a.shift) - 1) >> a.shift;           // len <= room: no overflow near 2^31 (width * page < 2^31)
    if (add < 0) { give = have; return; }
    if ((long)len + add > room) { bad |= 2; return; }
    more = add;
    need = (int)(((long)len + add + (1 << a.shift) - 1) >> a.shift) - have;
}

// Tables, ring and token rows of a step, spread over `nthr` threads of which this is `tid`.  len / take / give / start:
// per request (start has B + 1); head, count: the ring before the step.
__device__ void plan_fill(const PlanArgs& a, const int* len, const int* take, const int* give, const int* start, long tid, long nthr,
                          int head, int count, bool ok) {
    const int page = 1 << a.shift, total = ok ? start[a.B] : 0;
    for (long t = tid; t < a.max_tokens; t += nthr) {
        int slot = -1, pos = 0;
        if (t < total) {
            int lo = 0, hi = a.B;                                      // start[lo] <= t < start[hi]
            while (hi - lo > 1) {
                const int mid = (lo + hi) >> 1;
                if (start[mid] <= t) lo = mid; else hi = mid;
            }
            const int n = len[lo], have = (n + page - 1) >> a.shift;
            pos = n + ((int)t - start[lo]);
            const int j = pos >> a.shift;
            int p;
            if (j < have) p = a.table[lo * a.ld_table + j];
            else {
                unsigned at = (unsigned)head + take[lo] + (j - have);
                p = a.ring[at >= (unsigned)a.n_pages ? at - a.n_pages : at];
            }
            slot = (p << a.shift) + (pos & (page - 1));
        }
        a.slots[t] = slot;
        a.positions[t] = pos;
    }
    if (!ok) return;
    const int lane = tid & 63;
    for (long b = tid >> 6; b < a.B; b += nthr >> 6) {                 // a wave per request
        const int n = len[b], add = a.add[b], have = (n + page - 1) >> a.shift;
        int* row = a.table + b * a.ld_table;
        if (add < 0) {
            for (int j = lane; j < have; j += 64) {
                unsigned at = (unsigned)head + count + give[b] + j;    // count + pages given <= n_pages: below 2 n
                a.ring[at >= (unsigned)a.n_pages ? at - a.n_pages : at] = row[j];
            }
        } else {
            const int need = ((n + add + page - 1) >> a.shift) - have;
            for (int j = lane; j < need; j += 64) {
                unsigned at = (unsigned)head + take[b] + j;
                row[have + j] = a.ring[at >= (unsigned)a.n_pages ? at - a.n_pages : at];
            }
        }
    }
}

template <bool ONE>
__global__ __launch_bounds__(PLAN_THREADS) void paged_plan_scan_kernel(PlanArgs a) {
    __shared__ int part[3][16];
    __shared__ long red[3][16];
    __shared__ int s_bad;
    __shared__ int s_len[ONE ? PLAN_THREADS : 1], s_take[ONE ? PLAN_THREADS : 1], s_give[ONE ? PLAN_THREADS : 1], s_start[ONE ? PLAN_THREADS + 1 : 1];
    const int tid = threadIdx.x, lane = tid & 63, w = tid >> 6;
    const int head = a.pool[0], count = a.pool[1];
    if (tid == 0) s_bad = (head < 0 || head >= a.n_pages || count < 0 || count > a.n_pages) ? 8 : 0;
    __syncthreads();
    // totals first (nothing is written unless the whole step fits)
    int bad = 0;
    long sum[3] = {0, 0, 0};
    int len, need, give, more;
    for (int b = tid; b < a.B; b += PLAN_THREADS) {
        plan_request(a, b, len, need, give, more, bad);
        sum[0] += need; sum[1] += give; sum[2] += more;
    }
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
        for (int i = 0; i < PLAN_THREADS / 64; ++i) tot[q] += red[q][i];
    int st = s_bad;
    if (tot[0] > count) st |= 1;
    if (tot[2] > a.max_tokens) st |= 4;
    if (tot[1] + count > a.n_pages) st |= 8;
    const bool ok = st == 0;
    int carry[3] = {0, 0, 0};
    const int passes = ONE ? 1 : (a.B + PLAN_THREADS - 1) / PLAN_THREADS;
    for (int c = 0; c < passes; ++c) {
        const int b = c * PLAN_THREADS + tid;
        if (!ONE || c) plan_request(a, b, len, need, give, more, bad);
        else if (b >= a.B) len = need = give = more = 0;
        int v[3] = {need, give, more}, in[3];
#pragma unroll
        for (int q = 0; q < 3; ++q) {
            in[q] = wave_scan_incl(ok ? v[q] : 0, lane);
            if (lane == 63) part[q][w] = in[q];
        }
        __syncthreads();
        int ex[3];
#pragma unroll
        for (int q = 0; q < 3; ++q) {
            int base = carry[q], all = 0;
            for (int i = 0; i < PLAN_THREADS / 64; ++i) {
                const int u = part[q][i];
                if (i < w) base += u;
                all += u;
            }
            ex[q] = base + in[q] - (ok ? v[q] : 0);
            carry[q] += all;
        }
        if (b < a.B) {
            a.q_start[b] = ex[2];
            if (ONE) { s_len[tid] = len; s_take[tid] = ex[0]; s_give[tid] = ex[1]; s_start[tid] = ex[2]; }
            else { a.ws[b] = len; a.ws[a.B + b] = ex[0]; a.ws[2 * (long)a.B + b] = ex[1]; }
            if (ok) a.lens_out[b] = a.add[b] < 0 ? 0 : len + more;
            else if (a.lens_out != a.lens) a.lens_out[b] = a.lens[b];
        }
        __syncthreads();
    }
    if (tid == 0) {
        a.q_start[a.B] = carry[2];
        if (ONE) s_start[a.B] = carry[2];
        else { int* t = a.ws + 3 * (long)a.B; t[0] = head; t[1] = count; t[2] = ok; }
        a.status[0] = st;
        if (ok) {
            unsigned h = (unsigned)head + (unsigned)tot[0];
            a.pool_out[0] = h >= (unsigned)a.n_pages ? h - a.n_pages : h;
            a.pool_out[1] = count - (int)tot[0] + (int)tot[1];
        } else if (a.pool_out != a.pool) { a.pool_out[0] = head; a.pool_out[1] = count; }
    }
    if (ONE) {
        __syncthreads();
        plan_fill(a, s_len, s_take, s_give, s_start, tid, PLAN_THREADS, head, count, ok);
    }
}
__global__ __launch_bounds__(256) void paged_plan_fill_kernel(PlanArgs a) {
    const int* t = a.ws + 3 * (long)a.B;
    plan_fill(a, a.ws, a.ws + a.B, a.ws + 2 * (long)a.B, a.q_start, (long)blockIdx.x * 256 + threadIdx.x, (long)gridDim.x * 256, t[0], t[1], t[2]);
}

static inline int page_shift(int64_t page) {
    for (int s = 4; s <= 8; ++s)
        if (page == (1 << s)) return s;
    return -1;
}
static inline bool plan_one(int64_t B, int64_t max_tokens) { return B <= PLAN_THREADS && max_tokens <= PLAN_ONE; }

extern "C" int64_t avsr_paged_plan_workspace_bytes(int64_t B, int64_t max_tokens) {
    return plan_one(B, max_tokens) ? 0 : (3 * B + 4) * 4;
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
    if (!plan_one(B, max_tokens) && !workspace) return AVSR_EINVAL;
    PlanArgs a = {lens, add, table, (long)ld_table, (int)width, ring, (int)n_pages, pool, lens_out, pool_out, (int)B, shift, (int)max_tokens,
                  q_start, slots, positions, status, (int*)workspace};
    hipStream_t s = (hipStream_t)stream;
    if (plan_one(B, max_tokens)) hipLaunchKernelGGL(paged_plan_scan_kernel<true>, dim3(1), dim3(PLAN_THREADS), 0, s, a);
    else {
        hipLaunchKernelGGL(paged_plan_scan_kernel<false>, dim3(1), dim3(PLAN_THREADS), 0, s, a);
        int64_t blocks = (max_tokens + 255) / 256, more = (B + 3) / 4;
        blocks = blocks > more ? blocks : more;
        hipLaunchKernelGGL(paged_plan_fill_kernel, dim3((unsigned)(blocks < 2048 ? blocks : 2048)), dim3(256), 0, s, a);
    }
    return avsr_launch_status();
}

// ================================================================ write ====
// One 16-byte piece of a page per thread and turn; a row of the pages (one token and head) is 128 or more contiguous
// bytes.  Pure traffic: every byte is read once and written once.
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
    if ((ldk | ldv | k_head | v_head) % qi || (k_page_stride | k_head_stride | v_page_stride | v_head_stride) % qo ||
        ((uintptr_t)k | (uintptr_t)v | (uintptr_t)k_pages | (uintptr_t)v_pages) % 16) return AVSR_EUNSUPPORTED;
    if (rows == 0) return AVSR_OK;
    WriteArgs a = {k, v, ldk, ldv, k_head, v_head, k_pages, v_pages, k_page_stride, k_head_stride, v_page_stride, v_head_stride,
                   slots, rows, (int)H, head_dim == 64 ? 6 : 7, shift, n_pages << shift};
    const int64_t n = rows * 2 * H * head_dim / ((in_dtype == AVSR_F32 && page_dtype == AVSR_F32) ? 4 : 8);
    hipStream_t s = (hipStream_t)stream;
    const int64_t blocks = (n + 1023) / 1024;
    if (blocks > 0x7fffffff) return AVSR_EUNSUPPORTED;
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
    int splits, tiles_few, few_rows; float* part;  // few: key splits, row tiles per request; few_rows: largest request it takes (0 = any)
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
    // P rounds to bf16 for the product (half a step of 2^-8 relative each, averaged over the keys; the row sum stays fp32)
    static __device__ __forceinline__ bf16x8 probs(const f32x4 (&p)[2]) {
        bf16x8 b;
#pragma unroll
        for (int r = 0; r < 4; ++r) { b[r] = (bf16_t)p[0][r]; b[4 + r] = (bf16_t)p[1][r]; }
        return b;
    }
    static __device__ __forceinline__ void zero_key(V& v, int j) { v.x[j] = (vrow_t)(0u); }
    static __device__ __forceinline__ int key_of_v(int j, int g) { return 8 * g + j; }
    static __device__ __forceinline__ bool odd_value(const V& v) {       // any value that is not finite
        bool f = false;
#pragma unroll
        for (int j = 0; j < 8; ++j)
#pragma unroll
            for (int w = 0; w < VW / 2; ++w) f |= (v.x[j][w] & 0x7F80u) == 0x7F80u || (v.x[j][w] & 0x7F800000u) == 0x7F800000u;
        return f;
    }
    static __device__ __forceinline__ f32x4 pv(const V& v, int e, const f32x4 (&p)[2], f32x4 o) {
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(column(v, e), probs(p), o, 0, 0, 0);
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
    static __device__ __forceinline__ bool odd_value(const V& v) {
        bool f = false;
#pragma unroll
        for (int j = 0; j < 8; ++j)
#pragma unroll
            for (int w = 0; w < VW / 4; ++w)
#pragma unroll
                for (int x = 0; x < 4; ++x) f |= (__builtin_bit_cast(unsigned, v.x[j][w][x]) & 0x7F800000u) == 0x7F800000u;
        return f;
    }
    static __device__ __forceinline__ f32x4 pv(const V& v, int e, const f32x4 (&p)[2], f32x4 o) {
#pragma unroll
        for (int j = 0; j < 8; ++j) o = __builtin_amdgcn_mfma_f32_16x16x4f32(v.x[j][e >> 2][e & 3], p[j >> 2][j & 3], o, 0, 0, 0);
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
__device__ __forceinline__ TilePages tile_pages(const AttnArgs& a, const int* row, int kt, int kend) {
    TilePages t;
    const int last = (kend - 1) >> a.shift;                              // kend >= 1
    const int j = (kt * 32) >> a.shift;
    t.p0 = row[min(j, last)];
    t.p1 = a.shift == 4 ? row[min(j + 1, last)] : t.p0;
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
// largest of them over the wave's rows (a tile that ends at or before kmin needs no comparison).
template <typename F, int NT, int D>
__device__ __forceinline__ void attend_tile(State<NT, D>& st, const typename F::Q (&q)[NT], const typename F::K& k, typename F::V& v,
                                            const int (&limit)[NT], int kt, int kmin, int kmax, bool pages_ok, TilePages tp,
                                            const AttnArgs& a, int lane) {
    const int g = lane >> 4, k0 = kt * 32;
    const bool whole = pages_ok && k0 + 31 <= kmin;
    bool odd = false;
    if (!whole) {                                     // nothing a key beyond every row holds may reach the products
        const bool bad0 = (unsigned)tp.p0 >= (unsigned)a.n_pages, bad1 = (unsigned)tp.p1 >= (unsigned)a.n_pages;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const int key = F::key_of_v(j, g);
            if (k0 + key > kmax || ((key & 16) ? bad1 : bad0)) F::zero_key(v, j);
        }
        odd = __ballot(F::odd_value(v)) != 0;          // 0 * inf: a row's unseen keys need care
    }
#pragma unroll
    for (int n = 0; n < NT; ++n) {
        f32x4 s[2];
        F::scores(s, k, q[n]);
        if (!whole) {
            const bool bad0 = (unsigned)tp.p0 >= (unsigned)a.n_pages, bad1 = (unsigned)tp.p1 >= (unsigned)a.n_pages;
#pragma unroll
            for (int t = 0; t < 2; ++t)
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    const int key = F::key_of_score(t, r, g);
                    s[t][r] = (k0 + key > limit[n] || ((key & 16) ? bad1 : bad0)) ? -INFINITY : s[t][r] * a.c;
                }
        } else {
#pragma unroll
            for (int t = 0; t < 2; ++t)
#pragma unroll
                for (int r = 0; r < 4; ++r) s[t][r] *= a.c;
        }
        float mx = fmaxf(fmaxf(fmaxf(s[0][0], s[0][1]), fmaxf(s[0][2], s[0][3])), fmaxf(fmaxf(s[1][0], s[1][1]), fmaxf(s[1][2], s[1][3])));
        mx = fmaxf(st.m[n], max_over_groups(mx));
        if (__ballot(mx > st.m[n])) {                  // some row's maximum moved
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
        if (!odd) {
#pragma unroll
            for (int e = 0; e < D / 16; ++e) st.o[n][e] = F::pv(v, e, s, st.o[n][e]);
        } else {                                       // row by row, its unseen keys' values out of the product
            for (int r = 0; r < 16; ++r) {
                const int lim = __builtin_amdgcn_readlane(limit[n], r);
                typename F::V vr = v;
#pragma unroll
                for (int j = 0; j < 8; ++j)
                    if (k0 + F::key_of_v(j, g) > lim) F::zero_key(vr, j);
#pragma unroll
                for (int e = 0; e < D / 16; ++e) {
                    const f32x4 x = F::pv(vr, e, s, st.o[n][e]);
#pragma unroll
                    for (int y = 0; y < 4; ++y) st.o[n][e][y] = (lane & 15) == r ? x[y] : st.o[n][e][y];
                }
            }
        }
    }
}

// Tiles first, first + step, ... < end of the request's keys.  The next tile's keys and values are in flight while a
// tile is computed, its page numbers one tile further ahead.
template <typename F, typename T, int NT, int D>
__device__ __forceinline__ void attend(State<NT, D>& st, const AttnArgs& a, const typename F::Q (&q)[NT], const int (&limit)[NT],
                                       const int* row, int hk, int first, int step, int end, int kmin, int kmax, int lane) {
    if (first >= end) return;
    const int i = lane & 15, g = lane >> 4;
    typename F::K k[2];
    typename F::V v[2];
    TilePages tp[2], next;
    tp[0] = tile_pages(a, row, first, kmax + 1);
    load_tile<F, T>(a, k[0], v[0], tp[0], first, hk, i, g, D);
    next = tile_pages(a, row, min(first + step, end - 1), kmax + 1);
    auto one = [&](int kt, int cur) {
        if (kt + step < end) {
            tp[cur ^ 1] = next;
            load_tile<F, T>(a, k[cur ^ 1], v[cur ^ 1], next, kt + step, hk, i, g, D);
            next = tile_pages(a, row, min(kt + 2 * step, end - 1), kmax + 1);
        }
        const TilePages p = tp[cur];
        const bool ok = (unsigned)p.p0 < (unsigned)a.n_pages && (unsigned)p.p1 < (unsigned)a.n_pages;
        attend_tile<F, NT, D>(st, q, k[cur], v[cur], limit, kt, kmin, kmax, ok, p, a, lane);
    };
    for (int kt = first; kt < end; kt += 2 * step) {
        one(kt, 0);
        if (kt + step < end) one(kt + step, 1);
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

// ---- few rows: the four waves of a workgroup take every fourth tile of the keys and are merged through LDS; a split
// grid leaves {m, l, O} per row and split for paged_attn_join_kernel.
#define FEW_WAVES 4
template <typename T, int D>
__global__ __launch_bounds__(64 * FEW_WAVES) void paged_attn_few_kernel(AttnArgs a) {
    typedef Frag<T, D> F;
    __shared__ float s_m[FEW_WAVES][16], s_l[FEW_WAVES][16];
    __shared__ float s_o[FEW_WAVES][16][D + 4];
    const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int i = lane & 15, g = lane >> 4;
    const int split = blockIdx.x % a.splits, x = blockIdx.x / a.splits;
    const int hk = x % a.Hk, b = x / a.Hk;
    const Req r = request(a, b);
    const int rows = r.nq * a.G;
    if (a.few_rows && rows > a.few_rows) return;
    const int* row = a.table + b * a.ld_table;
    for (int r0 = blockIdx.y * 16; r0 < rows; r0 += gridDim.y * 16) {
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
        if (kmax >= 0) attend<F, T, 1, D>(st, a, q, limit, row, hk, t0 + w, FEW_WAVES, t1, kmin, kmax, lane);
        st.l[0] = xor_add<32>(xor_add<16>(st.l[0]));
        if (g == 0) { s_m[w][i] = st.m[0]; s_l[w][i] = st.l[0]; }
        if (i < n_rows) {
#pragma unroll
            for (int rr = 0; rr < 4; ++rr)
#pragma unroll
                for (int e = 0; e < D / 16; ++e) s_o[w][i][(D / 4) * g + (D / 16) * rr + e] = st.o[0][e][rr];
        }
        __syncthreads();
        // 16 columns a thread
        for (int c = threadIdx.x; c < n_rows * (D / 16); c += 64 * FEW_WAVES) {
            const int rw = c / (D / 16), d = (c % (D / 16)) * 16;
            float m = s_m[0][rw];
#pragma unroll
            for (int u = 1; u < FEW_WAVES; ++u) m = fmaxf(m, s_m[u][rw]);
            const float ref = m == -INFINITY ? 0.f : m;
            float l = 0.f, o[16];
#pragma unroll
            for (int j = 0; j < 16; ++j) o[j] = 0.f;
#pragma unroll
            for (int u = 0; u < FEW_WAVES; ++u) {
                const float f = __builtin_amdgcn_exp2f(s_m[u][rw] - ref);
                l = fmaf(f, s_l[u][rw], l);
#pragma unroll
                for (int j = 0; j < 16; ++j) o[j] = fmaf(f, s_o[u][rw][d + j], o[j]);
            }
            const int t = (r0 + rw) / a.G, h = hk * a.G + (r0 + rw) - t * a.G;
            if (a.splits == 1) {
                const float inv = l == 0.f ? 0.f : 1.f / l;
#pragma unroll
                for (int j = 0; j < 16; ++j) o[j] *= inv;
                store_vals<64>((T*)a.o + (long)(r.q0 + t) * a.ldo + (long)h * a.ho + d, o);
            } else {
                float* p = a.part + (((long)(r.q0 + t) * (a.Hk * a.G) + h) * a.splits + split) * (D + 4);
                store_vals<64>(p + 4 + d, o);
                if (d == 0) { p[0] = m; p[1] = l; }
            }
        }
        __syncthreads();
    }
}

// Joins the splits of a row: a wave per row, one or two columns a lane.
template <typename T, int D>
__global__ __launch_bounds__(256) void paged_attn_join_kernel(AttnArgs a) {
    const int lane = threadIdx.x & 63;
    const long H = (long)a.Hk * a.G, rows = H * a.N;
    const long x = (long)blockIdx.x * 4 + (threadIdx.x >> 6);
    if (x >= rows) return;
    const int t = (int)(x / H), h = (int)(x - t * H);
    // rows that no request of the few kernel owns were not written there: nothing of theirs is read or stored here
    int lo = 0, hi = a.B;
    if (t < a.q_start[0] || t >= a.q_start[a.B]) return;
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (a.q_start[mid] <= t) lo = mid; else hi = mid;
    }
    const Req r = request(a, lo);
    if (t < r.q0 || t >= r.q0 + r.nq || (a.few_rows && r.nq * a.G > a.few_rows)) return;
    const float* p = a.part + x * a.splits * (D + 4);
    float m = -INFINITY;
    for (int s = 0; s < a.splits; ++s) m = fmaxf(m, p[s * (D + 4)]);
    const float ref = m == -INFINITY ? 0.f : m;
    float l = 0.f, o[D / 64];
#pragma unroll
    for (int c = 0; c < D / 64; ++c) o[c] = 0.f;
    for (int s = 0; s < a.splits; ++s) {
        const float* ps = p + s * (D + 4);
        const float f = __builtin_amdgcn_exp2f(ps[0] - ref);
        l = fmaf(f, ps[1], l);
#pragma unroll
        for (int c = 0; c < D / 64; ++c) o[c] = fmaf(f, ps[4 + 64 * c + lane], o[c]);
    }
    const float inv = l == 0.f ? 0.f : 1.f / l;
    T* out = (T*)a.o + (long)t * a.ldo + (long)h * a.ho;
#pragma unroll
    for (int c = 0; c < D / 64; ++c) out[64 * c + lane] = from_f32<T>(o[c] * inv);
}

// ---- many rows: each of the four waves takes 16 NT rows of the tile and walks all of its keys.
template <typename T, int D, int NT>
__global__ __launch_bounds__(256) void paged_attn_chunk_kernel(AttnArgs a) {
    typedef Frag<T, D> F;
    constexpr int TR = 64 * NT;
    const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int i = lane & 15, g = lane >> 4;
    const int hk = blockIdx.x % a.Hk, tile = blockIdx.x / a.Hk;
    // request b owns the tiles from q_start[b]*G/TR + b on: at least one more than it fills
    int lo = 0, hi = a.B;
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if ((int)((long)a.q_start[mid] * a.G / TR) + mid <= tile) lo = mid; else hi = mid;
    }
    const Req r = request(a, lo);
    const int rows = r.nq * a.G;
    const int r0 = (tile - ((int)((long)a.q_start[lo] * a.G / TR) + lo)) * TR + w * 16 * NT;
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
    if (kmax >= 0) attend<F, T, NT, D>(st, a, q, limit, a.table + lo * a.ld_table, hk, 0, 1, (kmax >> 5) + 1, kmin, kmax, lane);
#pragma unroll
    for (int n = 0; n < NT; ++n) {
        const float l = xor_add<32>(xor_add<16>(st.l[n]));
        const float inv = l == 0.f ? 0.f : 1.f / l;
        if (16 * n + i >= n_rows) continue;
        const int my = r0 + 16 * n + i, tok = my / a.G, head = hk * a.G + my - tok * a.G;
        float o[D / 4];
#pragma unroll
        for (int rr = 0; rr < 4; ++rr)
#pragma unroll
            for (int e = 0; e < D / 16; ++e) o[(D / 16) * rr + e] = st.o[n][e][rr] * inv;
        store_vals<D>((T*)a.o + (long)(r.q0 + tok) * a.ldo + (long)head * a.ho + (D / 4) * g, o);
    }
}

// Requests of up to FEW_ROWS rows (tokens times the heads that share a kv head) go to the first kernel.
#define FEW_ROWS 64
struct AttnPlan { int splits, tiles_few, few_rows; bool few, chunk; long chunk_tiles; };
static AttnPlan attn_plan(int64_t N, int64_t B, int64_t Hk, int64_t G, int64_t max_q, int64_t max_k, int chunk_rows) {
    AttnPlan p;
    const int64_t rows = max_q * G;
    p.chunk = rows > FEW_ROWS;
    p.few = !(p.chunk && B == 1 && N * G > FEW_ROWS);          // one large request: nothing for the first kernel
    p.few_rows = p.chunk ? FEW_ROWS : 0;
    p.tiles_few = (int)((rows < FEW_ROWS ? rows : FEW_ROWS) + 15) / 16;
    const int64_t wgs = B * Hk * p.tiles_few;
    int64_t s = (1024 + wgs - 1) / wgs;
    const int64_t most = (max_k + 255) / 256;
    s = s < most ? s : most;
    p.splits = (int)(s < 1 ? 1 : s > 64 ? 64 : s);
    p.chunk_tiles = N * G / chunk_rows + B;
    return p;
}
#define CHUNK_NT 2
extern "C" int64_t avsr_paged_attn_workspace_bytes(int64_t N, int64_t B, int64_t Hq, int64_t Hk, int64_t head_dim, int64_t max_q,
                                                   int64_t max_k) {
    if (N <= 0 || B <= 0 || Hk <= 0 || Hq % Hk || max_q <= 0 || max_k <= 0) return 0;
    const AttnPlan p = attn_plan(N, B, Hk, Hq / Hk, max_q, max_k, 64 * CHUNK_NT);
    return p.few && p.splits > 1 ? N * Hq * p.splits * (head_dim + 4) * 4 : 0;
}

template <typename T, int D>
static int launch_attn(hipStream_t s, AttnArgs a, const AttnPlan& p) {
    const int few_rows = p.few_rows;
    if (p.few) {
        a.few_rows = few_rows;
        a.splits = p.splits;
        hipLaunchKernelGGL((paged_attn_few_kernel<T, D>), dim3((unsigned)((long)a.B * a.Hk * p.splits), p.tiles_few), dim3(64 * FEW_WAVES), 0, s, a);
        if (p.splits > 1) {
            const long rows = (long)a.N * a.Hk * a.G;
            hipLaunchKernelGGL((paged_attn_join_kernel<T, D>), dim3((unsigned)((rows + 3) / 4)), dim3(256), 0, s, a);
        }
    }
    if (p.chunk) {
        a.few_rows = p.few ? few_rows : 0;
        hipLaunchKernelGGL((paged_attn_chunk_kernel<T, D, CHUNK_NT>), dim3((unsigned)(p.chunk_tiles * a.Hk)), dim3(256), 0, s, a);
    }
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
    const int shift = page_shift(page);
    if (shift < 0 || (head_dim != 64 && head_dim != 128) || n_pages > (1LL << (30 - shift)) || width > (1LL << (30 - shift))) return AVSR_EUNSUPPORTED;
    const int64_t qm = dtype == AVSR_F32 ? 4 : 8;
    if ((ldq | q_head | k_page_stride | k_head_stride | v_page_stride | v_head_stride | ldo | o_head) % qm ||
        ((uintptr_t)q | (uintptr_t)k_pages | (uintptr_t)v_pages | (uintptr_t)o) % 16) return AVSR_EUNSUPPORTED;
    if (N > (1 << 28) || N * Hq > (1LL << 30) || B > (1 << 24) || B * Hk > (1LL << 24)) return AVSR_EUNSUPPORTED;
    if (N == 0) return AVSR_OK;
    const int64_t mq = max_q < N ? max_q : N, mk = max_k < width * page ? max_k : width * page;
    const AttnPlan p = attn_plan(N, B, Hk, Hq / Hk, mq, mk, 64 * CHUNK_NT);
    const int64_t need = p.few && p.splits > 1 ? N * Hq * p.splits * (head_dim + 4) * 4 : 0;
    if (need && (!workspace || workspace_bytes < need || (uintptr_t)workspace % 16)) return AVSR_EINVAL;
    if (p.chunk_tiles * Hk > 0x7fffffff) return AVSR_EUNSUPPORTED;
    AttnArgs a = {q, ldq, q_head, k_pages, v_pages, k_page_stride, k_head_stride, v_page_stride, v_head_stride, table, ld_table, (int)width,
                  lens, q_start, o, ldo, o_head, (int)B, (int)Hk, (int)(Hq / Hk), (int)N, shift, (int)n_pages, scale * LOG2E, causal != 0,
                  1, p.tiles_few, p.few_rows, (float*)workspace};
    hipStream_t s = (hipStream_t)stream;
    if (dtype == AVSR_BF16) return head_dim == 64 ? launch_attn<bf16_t, 64>(s, a, p) : launch_attn<bf16_t, 128>(s, a, p);
    return head_dim == 64 ? launch_attn<float, 64>(s, a, p) : launch_attn<float, 128>(s, a, p);
}
