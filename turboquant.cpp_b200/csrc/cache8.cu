// The 8-bit key/value cache: a step's rows into its pages (layout and codes: cache8.cuh).
//
//   tq_write8   bias + rotary encoding on the fused projection; queries to a buffer, keys and values as codes into the pages
#include "cache8.cuh"

TQ_DEFINE_LAST_ERROR

namespace {

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
    int nh, pairing, written;          // written: the heads this launch takes (the queries alone, or all)
};

template <typename TA, typename TB, int KEPT>
__global__ void __launch_bounds__(256) write8_kernel(const TA* __restrict__ qkv, const TB* __restrict__ bias, WriteArgs a, TA* __restrict__ q_out, Cache8 c) {
    tq_grid_wait();                    // everything below may read what the previous kernel wrote
    tq_grid_launch_dependents();
    const int lane = threadIdx.x & 31, j = blockIdx.y * (blockDim.x >> 5) + (threadIdx.x >> 5), heads = a.nh + 2 * c.nkv;
    if (j >= a.written) return;
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

}  // namespace

// qkv [T, (nh + 2 nkv) * hd]; bias as long as a row, or null; cos and sin [positions, hd / 2] float32, or null; q_out [T, nh, hd].
// max_q_len: the longest run (cu_seqlens, held [n_seqs]: device).  codes null: the queries only.  Rows behind cu_seqlens[n_seqs] are left alone.
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
    const WriteArgs a{cos_t, sin_t, positions, cu_seqlens, held, nh, pairing, codes != nullptr ? nh + 2 * nkv : nh};
    // a run of n rows touches at most (n + 14) / 16 + 1 blocks
    const int units = max_q_len == 1 ? 1 : (max_q_len + 14) / C8_BLOCK + 1, heads = a.written, warps = units * n_seqs >= 128 ? 8 : 2;
    const dim3 grid(units, (heads + warps - 1) / warps, n_seqs);
    TQ_DISPATCH(act_dtype, TA, TQ_DISPATCH(bias != nullptr ? bias_dtype : act_dtype, TB,
        if (max_q_len == 1) tq_launch(grid, warps * 32, 0, stream)(write8_kernel<TA, TB, 1>, (const TA*)qkv, (const TB*)bias, a, (TA*)q_out, c);
        else tq_launch(grid, warps * 32, 0, stream)(write8_kernel<TA, TB, 4>, (const TA*)qkv, (const TB*)bias, a, (TA*)q_out, c)));
    TQ_CHECK_LAUNCH("write8");
    return 0;
}
