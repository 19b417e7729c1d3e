// The 8-bit key/value cache: a step's rows into its pages, and attention over them (layout and codes: cache8.cuh).
//
//   tq_write8       bias + rotary encoding on the fused projection; queries to a buffer, keys and values as codes into the pages
//   tq_attention8   softmax(scale q.K) V over the cache, causal, with an optional window; the log2 of each row's denominator on the side
//   tq_weigh8       the softmax weights that every cached row received, added up over a step's rows and a key/value head's query heads
#include "cache8.cuh"

TQ_DEFINE_LAST_ERROR

namespace {

constexpr float LOG2E = 1.4426950408889634f;

// eight consecutive elements as float32
__device__ __forceinline__ void load8(const __nv_bfloat16* p, float (&f)[8]) {
    const uint4 v = *reinterpret_cast<const uint4*>(p);
    const uint32_t u[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) { f[2 * i] = __uint_as_float(u[i] << 16); f[2 * i + 1] = __uint_as_float(u[i] & 0xffff0000u); }
}
__device__ __forceinline__ void load8(const float* p, float (&f)[8]) {
    const float4 a = *reinterpret_cast<const float4*>(p), b = *reinterpret_cast<const float4*>(p + 4);
    f[0] = a.x; f[1] = a.y; f[2] = a.z; f[3] = a.w; f[4] = b.x; f[5] = b.y; f[6] = b.z; f[7] = b.w;
}
__device__ __forceinline__ void store8(__nv_bfloat16* p, const float (&f)[8]) {
    uint32_t u[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const __nv_bfloat162 h = __floats2bfloat162_rn(f[2 * i], f[2 * i + 1]);
        u[i] = *reinterpret_cast<const uint32_t*>(&h);
    }
    *reinterpret_cast<uint4*>(p) = make_uint4(u[0], u[1], u[2], u[3]);
}
__device__ __forceinline__ void store8(float* p, const float (&f)[8]) {
    *reinterpret_cast<float4*>(p) = make_float4(f[0], f[1], f[2], f[3]);
    *reinterpret_cast<float4*>(p + 4) = make_float4(f[4], f[5], f[6], f[7]);
}

// ---------------------------------------------------------------------------------------
// The writer.  A unit is the rows a sequence brings into one block of 16; a warp takes one head of it, query heads among them, so that
// nothing is shared between warps: the block's largest magnitude is one reduction over the warp's registers, and rows the block holds
// already are rounded again by the same warp when its byte grows.  An item is eight rotation pairs of a row: 16 elements, two 16-byte
// loads of bfloat16 and two 8-byte stores of codes.  KEPT items a lane stay in registers between the maximum and the codes (heads of up
// to 128); longer heads are loaded twice, the second time from the caches.
// Products and sums of the rotation are rounded one by one: the codes are then a function of the inputs that any float32 program can
// state, and a rounding to 4 bits never depends on which product was fused.
// ---------------------------------------------------------------------------------------
struct WriteArgs {
    const float *cos_t, *sin_t;
    const int *positions, *cu_seqlens, *held;
    int nh, pairing, n_seqs;
};

template <typename TA, typename TB, int KEPT>
__global__ void __launch_bounds__(256) write8_kernel(const TA* __restrict__ qkv, const TB* __restrict__ bias, WriteArgs a, TA* __restrict__ q_out, Cache8 c) {
    tq_grid_wait();                    // everything below may read what the previous kernel wrote
    tq_grid_launch_dependents();
    const int lane = threadIdx.x & 31, j = blockIdx.y * (blockDim.x >> 5) + (threadIdx.x >> 5), heads = a.nh + 2 * c.nkv;
    if (j >= heads) return;
    const int seq = blockIdx.z, t_begin = a.cu_seqlens[seq], run = a.cu_seqlens[seq + 1] - t_begin;
    const int place0 = a.held[seq];
    const int block_start = (place0 / C8_BLOCK + (int)blockIdx.x) * C8_BLOCK;       // the unit's block, as a place
    const int first = max(block_start, place0), rows = min(block_start + C8_BLOCK, place0 + run) - first;
    if (rows <= 0) return;
    const int t0 = t_begin + first - place0, hd = c.hd, half = hd >> 1, groups = half >> 3, items = rows * groups;
    const bool is_q = j < a.nh, rotated = j < a.nh + c.nkv && a.cos_t != nullptr;
    const size_t width = (size_t)heads * hd;
    const TA* src = qkv + (size_t)t0 * width + (size_t)j * hd;
    const TB* b_row = bias != nullptr ? bias + (size_t)j * hd : nullptr;

    // the item's 16 elements, rotated; lo: elements at ia.., hi: at ib..
    auto item = [&](int it, float (&lo)[8], float (&hi)[8]) {
        const int r = it / groups, i = (it - r * groups) * 8;
        const TA* row = src + (size_t)r * width;
        const int ia = a.pairing == 0 ? i : 2 * i, ib = a.pairing == 0 ? i + half : 2 * i + 8;
        load8(row + ia, lo);
        load8(row + ib, hi);
        if (b_row != nullptr) {
            float x[8], y[8];
            load8(b_row + ia, x);
            load8(b_row + ib, y);
#pragma unroll
            for (int e = 0; e < 8; ++e) { lo[e] += x[e]; hi[e] += y[e]; }
        }
        if (rotated) {
            const size_t at = (size_t)a.positions[t0 + r] * half + i;
            float cs[8], sn[8];
            load8(a.cos_t + at, cs);
            load8(a.sin_t + at, sn);
            if (a.pairing == 0) {
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    const float u = lo[e], v = hi[e];
                    lo[e] = __fsub_rn(__fmul_rn(u, cs[e]), __fmul_rn(v, sn[e]));
                    hi[e] = __fadd_rn(__fmul_rn(u, sn[e]), __fmul_rn(v, cs[e]));
                }
            } else {
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const float u = lo[2 * e], v = lo[2 * e + 1], x = hi[2 * e], y = hi[2 * e + 1];
                    lo[2 * e] = __fsub_rn(__fmul_rn(u, cs[e]), __fmul_rn(v, sn[e]));
                    lo[2 * e + 1] = __fadd_rn(__fmul_rn(u, sn[e]), __fmul_rn(v, cs[e]));
                    hi[2 * e] = __fsub_rn(__fmul_rn(x, cs[e + 4]), __fmul_rn(y, sn[e + 4]));
                    hi[2 * e + 1] = __fadd_rn(__fmul_rn(x, sn[e + 4]), __fmul_rn(y, cs[e + 4]));
                }
            }
        }
    };
    if (is_q) {
        TA* dst = q_out + ((size_t)t0 * a.nh + j) * hd;
        for (int it = lane; it < items; it += 32) {
            float lo[8], hi[8];
            item(it, lo, hi);
            const int r = it / groups, i = (it - r * groups) * 8;
            TA* d = dst + (size_t)r * a.nh * hd;
            store8(d + (a.pairing == 0 ? i : 2 * i), lo);
            store8(d + (a.pairing == 0 ? i + half : 2 * i + 8), hi);
        }
        return;
    }
    const int plane = j >= a.nh + c.nkv ? 1 : 0, g = j - a.nh - plane * c.nkv;
    const int page = c.page_of(seq, first), row0 = block_start % c.page_size, old = first - block_start;
    uint8_t* codes = c.codes + c.codes_at(page, plane, g) + (size_t)row0 * hd;
    uint8_t* byte = c.scales + c.scales_at(page, plane, g) + row0 / C8_BLOCK;
    const uint32_t was = old > 0 ? max((uint32_t)*byte, 1u) : 1u;
    float lo[KEPT][8], hi[KEPT][8];
    uint32_t top = 0;
    auto largest = [&](const float (&x)[8], const float (&y)[8]) {
#pragma unroll
        for (int e = 0; e < 8; ++e) top = max(top, max(c8_magnitude(x[e]), c8_magnitude(y[e])));
    };
    // one lane's items; a head too long for its registers goes through the first of them one by one
    const bool kept = items <= 32 * KEPT;
    if (kept) {
#pragma unroll
        for (int k = 0; k < KEPT; ++k)
            if (lane + 32 * k < items) { item(lane + 32 * k, lo[k], hi[k]); largest(lo[k], hi[k]); }
    } else {
        for (int it = lane; it < items; it += 32) { item(it, lo[0], hi[0]); largest(lo[0], hi[0]); }
    }
    top = __reduce_max_sync(0xffffffffu, top);
    const uint32_t b = max(c8_byte(top), was);
    const float inv = c8_inverse(b);
    auto write = [&](int it, const float (&x)[8], const float (&y)[8]) {
        const int r = it / groups, i = (it - r * groups) * 8;
        uint8_t* d = codes + (size_t)(old + r) * hd;
        uint32_t w[4];
#pragma unroll
        for (int e = 0; e < 2; ++e) {
            w[e] = c8_encode2(x[4 * e] * inv, x[4 * e + 1] * inv) | (c8_encode2(x[4 * e + 2] * inv, x[4 * e + 3] * inv) << 16);
            w[2 + e] = c8_encode2(y[4 * e] * inv, y[4 * e + 1] * inv) | (c8_encode2(y[4 * e + 2] * inv, y[4 * e + 3] * inv) << 16);
        }
        *reinterpret_cast<uint2*>(d + (a.pairing == 0 ? i : 2 * i)) = make_uint2(w[0], w[1]);
        *reinterpret_cast<uint2*>(d + (a.pairing == 0 ? i + half : 2 * i + 8)) = make_uint2(w[2], w[3]);
    };
    if (kept) {
#pragma unroll
        for (int k = 0; k < KEPT; ++k)
            if (lane + 32 * k < items) write(lane + 32 * k, lo[k], hi[k]);
    } else {
        for (int it = lane; it < items; it += 32) { item(it, lo[0], hi[0]); write(it, lo[0], hi[0]); }
    }
    if (b > was && old > 0) {
        const uint32_t factor = c8_shift_factor((int)min(b - was, 25u));
        for (int v = lane; v < old * (hd / 16); v += 32) {
            uint4* p = reinterpret_cast<uint4*>(codes) + v;
            *p = c8_shift16(*p, factor);
        }
    }
    if (lane == 0) *byte = (uint8_t)b;
}

// ---------------------------------------------------------------------------------------
// Attention, the plain way: a block per (row, query head), its warps share the keys, a lane holds every 32nd element.
// ---------------------------------------------------------------------------------------
template <typename TA>
__global__ void __launch_bounds__(128) attention8_kernel(const TA* __restrict__ q, Cache8 c, const int* __restrict__ cu_seqlens, const int* __restrict__ held,
                                                         int window, float scale, TA* __restrict__ out, float* __restrict__ lse, int nh) {
    tq_grid_wait();                    // everything below may read what the previous kernel wrote
    tq_grid_launch_dependents();
    constexpr int E = C8_MAX_HEAD_DIM / 32;
    __shared__ float s_o[4][C8_MAX_HEAD_DIM], s_m[4], s_l[4];
    const int seq = blockIdx.z, r = blockIdx.x, h = blockIdx.y, t_begin = cu_seqlens[seq];
    if (r >= cu_seqlens[seq + 1] - t_begin) return;
    const int t = t_begin + r, place = held[seq] + r, warp = threadIdx.x >> 5, lane = threadIdx.x & 31, hd = c.hd, g = h / (nh / c.nkv);
    float qv[E], o[E];
#pragma unroll
    for (int e = 0; e < E; ++e) {
        qv[e] = lane + 32 * e < hd ? tq_to_float(q[((size_t)t * nh + h) * hd + lane + 32 * e]) * (scale * LOG2E) : 0.f;
        o[e] = 0.f;
    }
    float m = -INFINITY, l = 0.f;
    for (int p = (window > 0 ? max(0, place + 1 - window) : 0) + warp; p <= place; p += 4) {
        const int page = c.page_of(seq, p), row = p % c.page_size;
        const uint8_t* k = c.codes + c.codes_at(page, 0, g) + (size_t)row * hd;
        const uint8_t* v = c.codes + c.codes_at(page, 1, g) + (size_t)row * hd;
        float s = 0.f;
#pragma unroll
        for (int e = 0; e < E; ++e) if (lane + 32 * e < hd) s += qv[e] * c8_float(k[lane + 32 * e]);
        s = tq_warp_sum(s) * c8_scale(c.scales[c.scales_at(page, 0, g) + row / C8_BLOCK]);
        const float mn = fmaxf(m, s), old = m == -INFINITY ? 0.f : exp2f(m - mn), w = exp2f(s - mn), sv = w * c8_scale(c.scales[c.scales_at(page, 1, g) + row / C8_BLOCK]);
        l = l * old + w;
#pragma unroll
        for (int e = 0; e < E; ++e) if (lane + 32 * e < hd) o[e] = o[e] * old + sv * c8_float(v[lane + 32 * e]);
        m = mn;
    }
#pragma unroll
    for (int e = 0; e < E; ++e) s_o[warp][lane + 32 * e] = o[e];
    if (lane == 0) { s_m[warp] = m; s_l[warp] = l; }
    __syncthreads();
    const float M = fmaxf(fmaxf(s_m[0], s_m[1]), fmaxf(s_m[2], s_m[3]));
    float f[4], L = 0.f;
#pragma unroll
    for (int w = 0; w < 4; ++w) { f[w] = s_m[w] == -INFINITY ? 0.f : exp2f(s_m[w] - M); L += f[w] * s_l[w]; }
    for (int d = threadIdx.x; d < hd; d += blockDim.x)
        out[((size_t)t * nh + h) * hd + d] = tq_from_float<TA>((s_o[0][d] * f[0] + s_o[1][d] * f[1] + s_o[2][d] * f[2] + s_o[3][d] * f[3]) / L);
    if (lse != nullptr && threadIdx.x == 0) lse[(size_t)t * nh + h] = M + log2f(L);
}

// Sums of weights, the plain way: a warp per cached row of a key/value head, which walks the step's rows that see it.  One writer per
// sum and a fixed order: the same bits every time.
template <typename TA>
__global__ void __launch_bounds__(128) weigh8_kernel(const TA* __restrict__ q, Cache8 c, const int* __restrict__ cu_seqlens, const int* __restrict__ held,
                                                     int window, float scale, const float* __restrict__ lse, float* __restrict__ weights, int nh) {
    tq_grid_wait();                    // everything below may read what the previous kernel wrote
    tq_grid_launch_dependents();
    constexpr int E = C8_MAX_HEAD_DIM / 32;
    const int seq = blockIdx.z, g = blockIdx.y, lane = threadIdx.x & 31, hd = c.hd, per = nh / c.nkv;
    const int p = blockIdx.x * 4 + (threadIdx.x >> 5), t_begin = cu_seqlens[seq], run = cu_seqlens[seq + 1] - t_begin, start = held[seq];
    if (run <= 0 || p >= start + run || (window > 0 && p + window <= start)) return;     // no row of the step sees it
    const int page = c.page_of(seq, p), row = p % c.page_size;
    const uint8_t* k = c.codes + c.codes_at(page, 0, g) + (size_t)row * hd;
    float kv[E];
    const float ks = c8_scale(c.scales[c.scales_at(page, 0, g) + row / C8_BLOCK]) * (scale * LOG2E);
#pragma unroll
    for (int e = 0; e < E; ++e) kv[e] = lane + 32 * e < hd ? c8_float(k[lane + 32 * e]) : 0.f;
    float sum = 0.f;
    for (int r = max(0, p - start); r < run && (window <= 0 || start + r - p < window); ++r)
        for (int h = g * per; h < (g + 1) * per; ++h) {
            const size_t at = (size_t)(t_begin + r) * nh + h;
            float s = 0.f;
#pragma unroll
            for (int e = 0; e < E; ++e) if (lane + 32 * e < hd) s += tq_to_float(q[at * hd + lane + 32 * e]) * kv[e];
            sum += exp2f(tq_warp_sum(s) * ks - lse[at]);
        }
    if (lane == 0) {
        float* w = weights + ((size_t)page * c.nkv + g) * c.page_size + row;
        *w = (p < start ? *w : 0.f) + sum;
    }
}

}  // namespace

// qkv [T, (nh + 2 nkv) * hd]; bias as long as a row, or null; cos and sin [positions, hd / 2] float32, or null; q_out [T, nh, hd].
// max_q_len: the longest run (cu_seqlens, held [n_seqs]: device).  Rows behind cu_seqlens[n_seqs] are left alone.
TQ_EXPORT int tq_write8(const void* qkv, int act_dtype, const void* bias, int bias_dtype, const float* cos_t, const float* sin_t, int pairing,
                        const int* positions, const int* cu_seqlens, const int* held, const int* page_table, int table_stride, int page_size,
                        void* q_out, void* codes, void* scales, int n_pages, int n_seqs, int max_q_len, int nh, int nkv, int hd, cudaStream_t stream) {
    if (n_seqs == 0 || max_q_len == 0) return 0;
    int rc = c8_check("write8", codes, scales, page_size, n_pages, nkv, hd, table_stride);
    if (rc) return rc;
    TQ_REQUIRE(nh >= 1 && nh % nkv == 0, "write8: %d heads are not a multiple of %d key/value heads", nh, nkv);
    TQ_REQUIRE((cos_t == nullptr) == (sin_t == nullptr), "write8: cos and sin tables come together");
    TQ_REQUIRE(n_seqs <= 65535 && max_q_len >= 1, "write8: %d sequences, longest run %d", n_seqs, max_q_len);
    TQ_REQUIRE(((uintptr_t)qkv | (uintptr_t)bias | (uintptr_t)q_out | (uintptr_t)cos_t | (uintptr_t)sin_t) % 16 == 0, "write8: tensors must be 16-byte aligned");
    const Cache8 c{(uint8_t*)codes, (uint8_t*)scales, page_table, table_stride, page_size, n_pages, nkv, hd};
    const WriteArgs a{cos_t, sin_t, positions, cu_seqlens, held, nh, pairing, n_seqs};
    // a run of n rows touches at most (n + 14) / 16 + 1 blocks
    const int units = max_q_len == 1 ? 1 : (max_q_len + 14) / C8_BLOCK + 1, heads = nh + 2 * nkv, warps = units * n_seqs >= 128 ? 8 : 2;
    const dim3 grid(units, (heads + warps - 1) / warps, n_seqs);
    TQ_DISPATCH(act_dtype, TA, TQ_DISPATCH(bias != nullptr ? bias_dtype : act_dtype, TB,
        if (max_q_len == 1) tq_launch(grid, warps * 32, 0, stream)(write8_kernel<TA, TB, 1>, (const TA*)qkv, (const TB*)bias, a, (TA*)q_out, c);
        else tq_launch(grid, warps * 32, 0, stream)(write8_kernel<TA, TB, 4>, (const TA*)qkv, (const TB*)bias, a, (TA*)q_out, c)));
    TQ_CHECK_LAUNCH("write8");
    return 0;
}

// q [T, nh, hd], out [T, nh * hd]; place i sees j <= i with window == 0 or i - j < window.  lse [T, nh] float32 or null.
TQ_EXPORT int tq_attention8(const void* q, const void* codes, const void* scales, int act_dtype, const int* cu_seqlens, const int* held,
                            const int* page_table, int table_stride, int page_size, int window, float scale, void* out, float* lse, int n_pages,
                            int n_seqs, int max_q_len, int nh, int nkv, int hd, cudaStream_t stream) {
    if (n_seqs == 0 || max_q_len == 0) return 0;
    int rc = c8_check("attention8", codes, scales, page_size, n_pages, nkv, hd, table_stride);
    if (rc) return rc;
    TQ_REQUIRE(nh >= 1 && nh % nkv == 0 && nh <= 65535, "attention8: %d heads are not a multiple of %d key/value heads", nh, nkv);
    TQ_REQUIRE(n_seqs <= 65535 && max_q_len >= 1 && window >= 0, "attention8: %d sequences, longest run %d, window %d", n_seqs, max_q_len, window);
    const Cache8 c{(uint8_t*)codes, (uint8_t*)scales, page_table, table_stride, page_size, n_pages, nkv, hd};
    TQ_DISPATCH(act_dtype, TA, tq_launch(dim3(max_q_len, nh, n_seqs), 128, 0, stream)(attention8_kernel<TA>, (const TA*)q, c, cu_seqlens, held, window, scale, (TA*)out, lse, nh));
    TQ_CHECK_LAUNCH("attention8");
    return 0;
}

// weights of places below held[s] grow by, those of the step's own rows become, the sum over the step's rows and the head's query heads of
// 2^(scale log2(e) q.k - lse).  max_kv_len: at least the longest held[s] + run.
TQ_EXPORT int tq_weigh8(const void* q, const void* codes, const void* scales, int act_dtype, const int* cu_seqlens, const int* held,
                        const int* page_table, int table_stride, int page_size, int window, float scale, const float* lse, float* weights, int n_pages,
                        int n_seqs, int max_kv_len, int nh, int nkv, int hd, cudaStream_t stream) {
    if (n_seqs == 0 || max_kv_len == 0) return 0;
    int rc = c8_check("weigh8", codes, scales, page_size, n_pages, nkv, hd, table_stride);
    if (rc) return rc;
    TQ_REQUIRE(nh >= 1 && nh % nkv == 0 && nkv <= 65535, "weigh8: %d heads are not a multiple of %d key/value heads", nh, nkv);
    TQ_REQUIRE(n_seqs <= 65535 && max_kv_len >= 1 && window >= 0, "weigh8: %d sequences, %d places, window %d", n_seqs, max_kv_len, window);
    const Cache8 c{(uint8_t*)codes, (uint8_t*)scales, page_table, table_stride, page_size, n_pages, nkv, hd};
    TQ_DISPATCH(act_dtype, TA, tq_launch(dim3((max_kv_len + 3) / 4, nkv, n_seqs), 128, 0, stream)(weigh8_kernel<TA>, (const TA*)q, c, cu_seqlens, held, window, scale, lse, weights, nh));
    TQ_CHECK_LAUNCH("weigh8");
    return 0;
}
