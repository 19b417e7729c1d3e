// The 8-bit key/value cache: a step's rows into its pages (layout and codes: cache8.cuh).
//
//   tq_write8   bias + rotary encoding on the fused projection; queries to a buffer, keys and values as codes into the pages
#include "cache8.cuh"

TQ_DEFINE_LAST_ERROR

namespace {

// Eight consecutive elements as float32, in pairs for the packed operations.
struct Eight { tq_f32x2 p[4]; };
// the same as they lie in memory
template <typename T> struct Raw;
template <> struct Raw<__nv_bfloat16> {
    uint4 v;
    __device__ __forceinline__ void load(const __nv_bfloat16* p) { v = *reinterpret_cast<const uint4*>(p); }
    __device__ __forceinline__ Eight wide() const {
        const uint32_t u[4] = {v.x, v.y, v.z, v.w};
        Eight r;
#pragma unroll
        for (int i = 0; i < 4; ++i) r.p[i] = tq_pack2(__uint_as_float(u[i] << 16), __uint_as_float(u[i] & 0xffff0000u));
        return r;
    }
};
template <> struct Raw<float> {
    float4 a, b;
    __device__ __forceinline__ void load(const float* p) { a = *reinterpret_cast<const float4*>(p); b = *reinterpret_cast<const float4*>(p + 4); }
    __device__ __forceinline__ Eight wide() const { return Eight{{tq_pack2(a.x, a.y), tq_pack2(a.z, a.w), tq_pack2(b.x, b.y), tq_pack2(b.z, b.w)}}; }
};
__device__ __forceinline__ Eight load8(const float* p) {
    Raw<float> r;
    r.load(p);
    return r.wide();
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
// pairs of a row: 16 elements, two 16-byte loads of bfloat16 and two 8-byte stores of codes; a thread has one item of a unit, so that all of its
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
    int nh, pairing, written, each;    // written: the heads this launch takes (the queries alone, or all); each: units a thread takes one after another
};

// Runs of many rows: a thread goes through the items of up to WRITE_EACH heads, so that the cosines and sines, twice the bytes of a bfloat16 item,
// are fetched once, and the next item is on its way while one is worked on (prompts above, heads a thread: one 33 us, two 27, three 25.7, four
// 25.5, six 26.8, eight 29.5; before, each head with its own cosines, 29.8).  Not where fewer than WRITE_FILL blocks would be left a turn.
constexpr int WRITE_EACH = 4, WRITE_FILL = 148 * 4;
constexpr int WRITE_THREADS = 256;

// HD: the head size, or 0 where it is known at the launch only.  Blocks an SM: of float32, whose items take twice the registers, 3 (4,096 rows of
// 28 + 4 + 4 heads: 30.5 us, with the bias asked for ahead 34, and 39 with four blocks).  The bias of bfloat16 is asked for ahead (prompts above: 25.7
// us, else 28).
template <typename TA, typename TB, bool RUNS, int HD>
__global__ void __launch_bounds__(WRITE_THREADS, RUNS ? HD == 128 && sizeof(TA) == 2 ? 4 : 3 : 1) write8_kernel(const TA* __restrict__ qkv, const TB* __restrict__ bias, WriteArgs a,
                                                                                                                 TA* __restrict__ q_out, Cache8 c, int threads_) {
    tq_grid_wait();                    // everything below may read what the previous kernel wrote
    tq_grid_launch_dependents();
    __shared__ float s_top[3][WRITE_THREADS / 32];
    const int hd = HD ? HD : c.hd, threads = !RUNS ? 32 : HD ? HD : threads_;
    const int unit = threadIdx.x / threads, it = threadIdx.x - unit * threads, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int side = RUNS && HD ? WRITE_THREADS / HD : blockDim.x / threads, warps = RUNS && HD ? WRITE_THREADS / 32 : blockDim.x / 32;
    const int each = RUNS ? a.each : 1, j0 = blockIdx.y * side * each, heads = a.nh + 2 * c.nkv;
    const int seq = blockIdx.z, t_begin = a.cu_seqlens[seq], run = a.cu_seqlens[seq + 1] - t_begin;
    const int place0 = a.held[seq];
    const int block_start = (place0 / C8_BLOCK + (int)blockIdx.x) * C8_BLOCK;       // the unit's block, as a place
    const int first = max(block_start, place0), rows = min(block_start + C8_BLOCK, place0 + run) - first;
    if (rows <= 0 || (!RUNS && j0 + unit >= a.written)) return;      // (runs: the whole block of threads returns or stays)
    const int t0 = t_begin + first - place0, half = hd >> 1, groups = half >> 3, items = rows * groups;
    const int r = it / groups, i = (it - r * groups) * 8;
    const int ia = a.pairing == 0 ? i : 2 * i, ib = a.pairing == 0 ? i + half : 2 * i + 8;       // where the item's two halves lie in the head
    const int row0 = c.row(block_start), old = first - block_start;
    const TA* row = qkv + (size_t)(t0 + r) * heads * hd;
    const bool inside = it < items;
    Raw<TA> next_lo = {}, next_hi = {};
    constexpr bool AHEAD = sizeof(TA) + sizeof(TB) == 4;             // the bias too
    Raw<TB> bias_lo = {}, bias_hi = {};
    auto ask = [&](int j) {
        if (!inside || j >= a.written) return;
        next_lo.load(row + j * hd + ia);
        next_hi.load(row + j * hd + ib);
        if (AHEAD && bias != nullptr) { bias_lo.load(bias + j * hd + ia); bias_hi.load(bias + j * hd + ib); }
    };
    ask(j0 + unit);
    const int page = a.written > a.nh ? c.page_of(seq, first) : 0;
    Eight cs = {}, sn = {};
    if (inside && j0 + unit < a.nh + c.nkv && a.cos_t != nullptr) {
        const size_t at = (size_t)a.positions[t0 + r] * half + i;
        cs = load8(a.cos_t + at);
        sn = load8(a.sin_t + at);
    }
    for (int k = 0; k < each; ++k) {
        const int j = j0 + k * side + unit;
        if (RUNS && j0 + k * side >= a.written) break;
        const bool mine = inside && j < a.written, is_q = j < a.nh;
        // where the unit's codes go, and the byte of rows the block holds already
        const int plane = j >= a.nh + c.nkv ? 1 : 0, g = j - a.nh - plane * c.nkv;
        uint8_t *codes = nullptr, *byte = nullptr;
        uint32_t was = 1;
        if (!is_q && j < a.written) {
            codes = c.codes + c.codes_at(page, plane, g) + (size_t)row0 * hd;
            byte = c.scales + c.scales_at(page, plane, g) + row0 / C8_BLOCK;
            if (old > 0) was = max((uint32_t)*byte, 1u);              // (by all of the unit's threads before one of them writes it)
        }
        Eight lo = next_lo.wide(), hi = next_hi.wide();
        if (bias != nullptr && mine) {
            Raw<TB> bias0 = bias_lo, bias1 = bias_hi;
            if (!AHEAD) { bias0.load(bias + j * hd + ia); bias1.load(bias + j * hd + ib); }
            const Eight x = bias0.wide(), y = bias1.wide();
#pragma unroll
            for (int e = 0; e < 4; ++e) { lo.p[e] = tq_add2(lo.p[e], x.p[e]); hi.p[e] = tq_add2(hi.p[e], y.p[e]); }
        }
        if (RUNS && k + 1 < each) ask(j + side);                      // on its way while this one is worked on
        if (mine) {
            if (j < a.nh + c.nkv && a.cos_t != nullptr) {
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
        // queries only (runs: all of the block's units, since the others' reductions are the block's)
        if (RUNS ? min(j0 + (k + 1) * side, a.written) <= a.nh : is_q) continue;
        // over the unit's threads; most: over the block's, where a block is several warps
        float most;
        auto over_unit = [&](float top, float* tops) {
            top = __uint_as_float(__reduce_max_sync(0xffffffffu, __float_as_uint(top)));       // magnitudes: ordered as integers are
            most = top;
            if (RUNS) {
                if (lane == 0) tops[warp] = top;
                __syncthreads();
                for (int w = 0; w < warps; ++w) most = fmaxf(most, tops[w]);
                for (int w = unit * (threads / 32); w < (unit + 1) * (threads / 32); ++w) top = fmaxf(top, tops[w]);
            }
            return top;
        };
        float top = over_unit(mine ? magnitude8(hi, magnitude8(lo, 0.f)) : 0.f, s_top[k & 1]);       // (s_top's other half is read until the next barrier)
        const bool infinite = top == INFINITY;
        if (most == INFINITY) {
            const float finite = over_unit(mine ? finite8(hi, finite8(lo, 0.f)) : 0.f, s_top[2]);
            if (infinite) top = finite;
        }
        if (codes == nullptr) continue;
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
    WriteArgs a{cos_t, sin_t, x.positions, x.cu_seqlens, x.held, nh, x.pairing, codes != nullptr ? nh + 2 * nkv : nh, 1};
    // a run of n rows touches at most (n + 14) / 16 + 1 blocks
    const bool runs = max_q_len > 1;
    const int units = runs ? (max_q_len + 14) / C8_BLOCK + 1 : 1, threads = runs ? (hd + 31) / 32 * 32 : 32;
    const int side = runs ? WRITE_THREADS / threads : n_seqs >= 32 ? 8 : 2;              // units a block takes side by side
    const long long blocks = (long long)units * ((a.written + side - 1) / side) * n_seqs;
    a.each = runs ? (int)max(1ll, min((long long)WRITE_EACH, blocks / WRITE_FILL)) : 1;
    const dim3 grid(units, (a.written + side * a.each - 1) / (side * a.each), n_seqs);
    TQ_DISPATCH(x.act_dtype, TA, TQ_DISPATCH(bias != nullptr ? x.bias_dtype : x.act_dtype, TB,
        auto kernel = runs ? (hd == 128 ? write8_kernel<TA, TB, true, 128> : hd == 64 ? write8_kernel<TA, TB, true, 64> : write8_kernel<TA, TB, true, 0>)
                           : (hd == 128 ? write8_kernel<TA, TB, false, 128> : write8_kernel<TA, TB, false, 0>);
        tq_launch(grid, side * threads, 0, x.stream)(kernel, (const TA*)qkv, (const TB*)bias, a, (TA*)x.q_out, c, threads)));
    TQ_CHECK_LAUNCH("write8");
    return 0;
}
