// The 8-bit key/value cache: a step's rows into its pages (layout and codes: cache8.cuh).
//
//   tq_write8   bias + rotary encoding on the fused projection; queries to a buffer, keys and values as codes into the pages
#include "cache8.cuh"

TQ_DEFINE_LAST_ERROR

namespace {

// Eight consecutive elements as float32, in pairs for the packed operations.
struct Eight { tq_f32x2 p[4]; };
__device__ __forceinline__ Eight load8(const __nv_bfloat16* p) {
    const uint4 v = *reinterpret_cast<const uint4*>(p);
    const uint32_t u[4] = {v.x, v.y, v.z, v.w};
    Eight r;
#pragma unroll
    for (int i = 0; i < 4; ++i) r.p[i] = tq_pack2(__uint_as_float(u[i] << 16), __uint_as_float(u[i] & 0xffff0000u));
    return r;
}
__device__ __forceinline__ Eight load8(const float* p) {
    const float4 a = *reinterpret_cast<const float4*>(p), b = *reinterpret_cast<const float4*>(p + 4);
    return Eight{{tq_pack2(a.x, a.y), tq_pack2(a.z, a.w), tq_pack2(b.x, b.y), tq_pack2(b.z, b.w)}};
}
__device__ __forceinline__ void store8(__nv_bfloat16* p, const Eight& f) {
    uint32_t u[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float2 x = tq_unpack2(f.p[i]);
        const __nv_bfloat162 h = __floats2bfloat162_rn(x.x, x.y);
        u[i] = *reinterpret_cast<const uint32_t*>(&h);
    }
    *reinterpret_cast<uint4*>(p) = make_uint4(u[0], u[1], u[2], u[3]);
}
__device__ __forceinline__ void store8(float* p, const Eight& f) {
    const float2 a = tq_unpack2(f.p[0]), b = tq_unpack2(f.p[1]), c = tq_unpack2(f.p[2]), d = tq_unpack2(f.p[3]);
    *reinterpret_cast<float4*>(p) = make_float4(a.x, a.y, b.x, b.y);
    *reinterpret_cast<float4*>(p + 4) = make_float4(c.x, c.y, d.x, d.y);
}
// the larger of `top` and the magnitudes of eight elements; NaN does not count
__device__ __forceinline__ float magnitude8(const Eight& f, float top) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float2 x = tq_unpack2(f.p[i]);
        asm("max.f32 %0, %1, %2, %3;" : "=f"(top) : "f"(top), "f"(fabsf(x.x)), "f"(fabsf(x.y)));
    }
    return top;
}
// the same over the finite elements alone
__device__ __forceinline__ float finite8(const Eight& f, float top) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float2 x = tq_unpack2(f.p[i]);
        top = fmaxf(top, fmaxf(__uint_as_float(c8_magnitude(x.x)), __uint_as_float(c8_magnitude(x.y))));
    }
    return top;
}
// eight elements as codes; infinite: some of the unit's elements may be (the conversion makes NaN of NaN, but 448 of them)
__device__ __forceinline__ uint2 encode8(const Eight& f, tq_f32x2 inv, bool infinite) {
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float2 x = tq_unpack2(tq_mul2(f.p[i], inv));
        uint16_t d;
        asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(d) : "f"(x.y), "f"(x.x));
        w[i] = d;
        if (infinite) w[i] = c8_encode2(x.x, x.y);
    }
    return make_uint2(__byte_perm(w[0], w[1], 0x5410), __byte_perm(w[2], w[3], 0x5410));
}

// ---------------------------------------------------------------------------------------
// The writer.  A unit is the rows a sequence brings into one block of 16, of one head, query heads among them.  An item is eight rotation
// pairs of a row: 16 elements, two 16-byte loads of bfloat16 and two 8-byte stores of codes; a thread has one item, so that all of a unit's
// loads are under way at once, and keeps it in registers between the block's largest magnitude (a reduction over the unit's threads) and
// its codes.  Rows the block holds already are rounded again by the same threads when its byte grows.
// Single tokens (RUNS false): a warp per unit.  Runs: head size threads per unit, rounded up to warps, so a thread for each of a whole
// block's items.  A warp per unit there too, four items a lane in 103 registers, took 42 us for prompts of 682 + 1,365 + 2,049 tokens,
// 16 + 16 + 16 heads of 128.
// Products and sums of the rotation are rounded one by one: the codes are then a function of the inputs that any float32 program can
// state, and a rounding to 4 bits never depends on which product was fused.
// ---------------------------------------------------------------------------------------
struct WriteArgs {
    const float *cos_t, *sin_t;
    const int *positions, *cu_seqlens, *held;
    int nh, pairing, written;          // written: the heads this launch takes (the queries alone, or all)
};

constexpr int WRITE_THREADS = 256;      // (512: 35 us for the prompts above, 31.5; five blocks an SM instead of four: 29.8)

// HD: the head size, or 0 where it is known at the launch only
template <typename TA, typename TB, bool RUNS, int HD>
__global__ void __launch_bounds__(WRITE_THREADS, RUNS && HD ? 5 : 1) write8_kernel(const TA* __restrict__ qkv, const TB* __restrict__ bias, WriteArgs a, TA* __restrict__ q_out, Cache8 c,
                                                               int threads_) {
    tq_grid_wait();                    // everything below may read what the previous kernel wrote
    tq_grid_launch_dependents();
    __shared__ float s_top[WRITE_THREADS / 32];
    const int hd = HD ? HD : c.hd, threads = !RUNS ? 32 : HD ? HD : threads_;
    const int unit = threadIdx.x / threads, it = threadIdx.x - unit * threads, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int j = blockIdx.y * (blockDim.x / threads) + unit, heads = a.nh + 2 * c.nkv;
    const int seq = blockIdx.z, t_begin = a.cu_seqlens[seq], run = a.cu_seqlens[seq + 1] - t_begin;
    const int place0 = a.held[seq];
    const int block_start = (place0 / C8_BLOCK + (int)blockIdx.x) * C8_BLOCK;       // the unit's block, as a place
    const int first = max(block_start, place0), rows = min(block_start + C8_BLOCK, place0 + run) - first;
    if (rows <= 0 || (!RUNS && j >= a.written)) return;              // (runs: the whole block of threads returns or stays)
    const int t0 = t_begin + first - place0, half = hd >> 1, groups = half >> 3, items = rows * groups;
    const bool mine = it < items && j < a.written, is_q = j < a.nh;
    const int r = it / groups, i = (it - r * groups) * 8;
    const int ia = a.pairing == 0 ? i : 2 * i, ib = a.pairing == 0 ? i + half : 2 * i + 8;       // where the item's two halves lie in the head
    // where the unit's codes go, and the byte of rows the block holds already, looked up beside the loads of the rows
    const int plane = j >= a.nh + c.nkv ? 1 : 0, g = j - a.nh - plane * c.nkv, row0 = c.row(block_start), old = first - block_start;
    uint8_t *codes = nullptr, *byte = nullptr;
    uint32_t was = 1;
    if (!is_q && j < a.written) {
        const int page = c.page_of(seq, first);
        codes = c.codes + c.codes_at(page, plane, g) + (size_t)row0 * hd;
        byte = c.scales + c.scales_at(page, plane, g) + row0 / C8_BLOCK;
        if (old > 0) was = max((uint32_t)*byte, 1u);                  // (by all of the unit's threads before one of them writes it)
    }
    Eight lo = {}, hi = {};
    if (mine) {
        const TA* row = qkv + ((size_t)(t0 + r) * heads + j) * hd;
        const bool rotated = j < a.nh + c.nkv && a.cos_t != nullptr;
        lo = load8(row + ia);
        hi = load8(row + ib);
        Eight cs = {}, sn = {};
        if (rotated) {
            const size_t at = (size_t)a.positions[t0 + r] * half + i;
            cs = load8(a.cos_t + at);
            sn = load8(a.sin_t + at);
        }
        if (bias != nullptr) {
            const Eight x = load8(bias + (size_t)j * hd + ia), y = load8(bias + (size_t)j * hd + ib);
#pragma unroll
            for (int e = 0; e < 4; ++e) { lo.p[e] = tq_add2(lo.p[e], x.p[e]); hi.p[e] = tq_add2(hi.p[e], y.p[e]); }
        }
        if (rotated) {
            // interleaved: the pairs' first elements together and their second ones, and back
            auto sort = [](Eight& x, Eight& y) {
                const float2 p[8] = {tq_unpack2(x.p[0]), tq_unpack2(x.p[1]), tq_unpack2(x.p[2]), tq_unpack2(x.p[3]),
                                     tq_unpack2(y.p[0]), tq_unpack2(y.p[1]), tq_unpack2(y.p[2]), tq_unpack2(y.p[3])};
#pragma unroll
                for (int e = 0; e < 4; ++e) { x.p[e] = tq_pack2(p[2 * e].x, p[2 * e + 1].x); y.p[e] = tq_pack2(p[2 * e].y, p[2 * e + 1].y); }
            };
            if (a.pairing != 0) sort(lo, hi);
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                // (the packed product and sum came out fused, their .rn notwithstanding)
                const float2 u = tq_unpack2(lo.p[e]), v = tq_unpack2(hi.p[e]), x = tq_unpack2(cs.p[e]), y = tq_unpack2(sn.p[e]);
                lo.p[e] = tq_pack2(__fsub_rn(__fmul_rn(u.x, x.x), __fmul_rn(v.x, y.x)), __fsub_rn(__fmul_rn(u.y, x.y), __fmul_rn(v.y, y.y)));
                hi.p[e] = tq_pack2(__fadd_rn(__fmul_rn(u.x, y.x), __fmul_rn(v.x, x.x)), __fadd_rn(__fmul_rn(u.y, y.y), __fmul_rn(v.y, x.y)));
            }
            if (a.pairing != 0) {
                const Eight u = lo, v = hi;
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const float2 x = tq_unpack2(u.p[e]), y = tq_unpack2(v.p[e]);
                    Eight& to = e < 2 ? lo : hi;
                    to.p[2 * (e & 1)] = tq_pack2(x.x, y.x);
                    to.p[2 * (e & 1) + 1] = tq_pack2(x.y, y.y);
                }
            }
        }
        if (is_q) {
            TA* d = q_out + ((size_t)(t0 + r) * a.nh + j) * hd;
            store8(d + ia, lo);
            store8(d + ib, hi);
        }
    }
    if (a.written == a.nh) return;                                    // queries only
    // over the unit's threads
    auto over_unit = [&](float top) {
        top = __uint_as_float(__reduce_max_sync(0xffffffffu, __float_as_uint(top)));       // magnitudes: ordered as integers are
        if (RUNS) {
            if (lane == 0) s_top[warp] = top;
            __syncthreads();
            for (int w = unit * (threads / 32); w < (unit + 1) * (threads / 32); ++w) top = fmaxf(top, s_top[w]);
        }
        return top;
    };
    float top = over_unit(magnitude8(hi, magnitude8(lo, 0.f)));
    const bool infinite = top == INFINITY;
    if (RUNS ? __syncthreads_or(infinite) : infinite) {
        const float finite = over_unit(finite8(hi, finite8(lo, 0.f)));
        if (infinite) top = finite;
    }
    if (codes == nullptr) return;
    const uint32_t b = max(c8_byte(__float_as_uint(top)), was);
    if (mine) {
        const float inv = c8_inverse(b);
        uint8_t* d = codes + (size_t)(old + r) * hd;
        *reinterpret_cast<uint2*>(d + ia) = encode8(lo, tq_pack2(inv, inv), infinite);
        *reinterpret_cast<uint2*>(d + ib) = encode8(hi, tq_pack2(inv, inv), infinite);
    }
    if (b > was && old > 0) {
        const uint32_t factor = c8_shift_factor((int)min(b - was, 25u));
        for (int v = it; v < old * (hd / 16); v += threads) {
            uint4* p = reinterpret_cast<uint4*>(codes) + v;
            *p = c8_shift16(*p, factor);
        }
    }
    if (it == 0) *byte = (uint8_t)b;
}

}  // namespace

// qkv [T, (nh + 2 nkv) * hd]; bias as long as a row, or null; cos and sin [positions, hd / 2] float32, or null; q_out [T, nh, hd].
// max_q_len: the longest run (cu_seqlens, held [n_seqs]: device).  codes null: the queries only.  Rows behind cu_seqlens[n_seqs] are left alone.
struct Write8Call {
    const void *qkv, *bias;
    const float *cos_t, *sin_t;
    const int *positions, *cu_seqlens, *held, *page_table;
    void *q_out, *codes, *scales;
    cudaStream_t stream;
    int act_dtype, bias_dtype, pairing, table_stride, page_size, n_pages, n_seqs, max_q_len, nh, nkv, hd;
};
TQ_EXPORT int tq_write8(const void* packed) {
    const Write8Call x = c8_call<Write8Call>(packed);
    const void *qkv = x.qkv, *bias = x.bias, *codes = x.codes, *scales = x.scales;
    const float *cos_t = x.cos_t, *sin_t = x.sin_t;
    const int page_size = x.page_size, n_pages = x.n_pages, n_seqs = x.n_seqs, max_q_len = x.max_q_len, nh = x.nh, nkv = x.nkv, hd = x.hd;
    if (n_seqs == 0 || max_q_len == 0) return 0;
    int rc = c8_check("write8", codes, scales, page_size, n_pages, nkv, hd, x.table_stride);
    if (rc) return rc;
    TQ_REQUIRE(nh >= 1 && nh % nkv == 0, "write8: %d heads are not a multiple of %d key/value heads", nh, nkv);
    TQ_REQUIRE((cos_t == nullptr) == (sin_t == nullptr), "write8: cos and sin tables come together");
    TQ_REQUIRE(n_seqs <= 65535 && max_q_len >= 1, "write8: %d sequences, longest run %d", n_seqs, max_q_len);
    TQ_REQUIRE(((uintptr_t)qkv | (uintptr_t)bias | (uintptr_t)x.q_out | (uintptr_t)cos_t | (uintptr_t)sin_t) % 16 == 0, "write8: tensors must be 16-byte aligned");
    const Cache8 c = c8_cache(codes, scales, x.page_table, x.table_stride, page_size, n_pages, nkv, hd);
    const WriteArgs a{cos_t, sin_t, x.positions, x.cu_seqlens, x.held, nh, x.pairing, codes != nullptr ? nh + 2 * nkv : nh};
    // a run of n rows touches at most (n + 14) / 16 + 1 blocks
    const bool runs = max_q_len > 1;
    const int units = runs ? (max_q_len + 14) / C8_BLOCK + 1 : 1, threads = runs ? (hd + 31) / 32 * 32 : 32;
    const int side = runs ? WRITE_THREADS / threads : n_seqs >= 32 ? 8 : 2;              // units a block takes side by side
    const dim3 grid(units, (a.written + side - 1) / side, n_seqs);
    TQ_DISPATCH(x.act_dtype, TA, TQ_DISPATCH(bias != nullptr ? x.bias_dtype : x.act_dtype, TB,
        auto kernel = runs ? (hd == 128 ? write8_kernel<TA, TB, true, 128> : hd == 64 ? write8_kernel<TA, TB, true, 64> : write8_kernel<TA, TB, true, 0>)
                           : (hd == 128 ? write8_kernel<TA, TB, false, 128> : write8_kernel<TA, TB, false, 0>);
        tq_launch(grid, side * threads, 0, x.stream)(kernel, (const TA*)qkv, (const TB*)bias, a, (TA*)x.q_out, c, threads)));
    TQ_CHECK_LAUNCH("write8");
    return 0;
}
