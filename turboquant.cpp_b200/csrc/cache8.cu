// The 8-bit key/value cache: a step's rows into its pages (layout and codes: cache8.cuh).
//
//   tq_write8   bias + rotary encoding on the fused projection; queries to a buffer, keys and values as codes into the pages
#include "cache8.cuh"

TQ_DEFINE_LAST_ERROR

namespace {

// Eight consecutive elements as they lie in memory, and as float32.  (Additions and products of pairs, as packed operations: 22.7 us,
// single ones 23.0, for the prompts below; 2.26 and 2.09 for a token; 3.6 and 3.3 for four prompts of up to 1,000 rows, 16 + 4 + 4 heads of 64.)
struct Eight { float v[8]; };
template <typename T> struct Raw;
template <> struct Raw<__nv_bfloat16> {
    uint4 v;
    __device__ __forceinline__ void load(const __nv_bfloat16* p) { v = *reinterpret_cast<const uint4*>(p); }
    __device__ __forceinline__ Eight wide() const {
        const uint32_t u[4] = {v.x, v.y, v.z, v.w};
        Eight r;
#pragma unroll
        for (int i = 0; i < 4; ++i) { r.v[2 * i] = __uint_as_float(u[i] << 16); r.v[2 * i + 1] = __uint_as_float(u[i] & 0xffff0000u); }
        return r;
    }
};
template <> struct Raw<float> {
    float4 a, b;
    __device__ __forceinline__ void load(const float* p) { a = *reinterpret_cast<const float4*>(p); b = *reinterpret_cast<const float4*>(p + 4); }
    __device__ __forceinline__ Eight wide() const { return Eight{{a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w}}; }
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
        const __nv_bfloat162 h = __floats2bfloat162_rn(f.v[2 * i], f.v[2 * i + 1]);
        u[i] = *reinterpret_cast<const uint32_t*>(&h);
    }
    *reinterpret_cast<uint4*>(p) = make_uint4(u[0], u[1], u[2], u[3]);
}
__device__ __forceinline__ void store8(float* p, const Eight& f) {
    *reinterpret_cast<float4*>(p) = make_float4(f.v[0], f.v[1], f.v[2], f.v[3]);
    *reinterpret_cast<float4*>(p + 4) = make_float4(f.v[4], f.v[5], f.v[6], f.v[7]);
}
// the larger of `top` and the magnitudes of eight elements; NaN does not count
__device__ __forceinline__ float magnitude8(const Eight& f, float top) {
#pragma unroll
    for (int i = 0; i < 8; i += 2) asm("max.f32 %0, %1, %2, %3;" : "=f"(top) : "f"(top), "f"(fabsf(f.v[i])), "f"(fabsf(f.v[i + 1])));
    return top;
}
// the same over the finite elements alone
__device__ __forceinline__ float finite8(const Eight& f, float top) {
#pragma unroll
    for (int i = 0; i < 8; ++i) top = fmaxf(top, __uint_as_float(c8_magnitude(f.v[i])));
    return top;
}
// eight elements as codes; INFINITE: some may be infinite (the conversion makes NaN of NaN, but 448 of them)
template <bool INFINITE> __device__ __forceinline__ uint2 encode8(const Eight& f, float inv) {
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float x = f.v[2 * i] * inv, y = f.v[2 * i + 1] * inv;
        if constexpr (INFINITE) w[i] = c8_encode2(x, y);
        else {
            uint16_t d;
            asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(d) : "f"(y), "f"(x));
            w[i] = d;
        }
    }
    return make_uint2(__byte_perm(w[0], w[1], 0x5410), __byte_perm(w[2], w[3], 0x5410));
}
// products and sums rounded one by one
__device__ __forceinline__ void rotate(float& u, float& v, float cs, float sn) {
    const float x = __fsub_rn(__fmul_rn(u, cs), __fmul_rn(v, sn));
    v = __fadd_rn(__fmul_rn(u, sn), __fmul_rn(v, cs));
    u = x;
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
    int nh, written, each;    // written: the heads this launch takes (the queries alone, or all); each: units a thread takes one after another
};

// Runs of many rows: a thread goes through the items of up to WRITE_EACH heads, so that the cosines and sines, twice the bytes of a bfloat16 item,
// are fetched once, and the next item is on its way while one is worked on (prompts above, heads a thread: one 33 us, two 27, three 25.7, four
// 25.5, six 26.8, eight 29.5).  Not where fewer than WRITE_FILL blocks would be left a turn.  Then 23.0, with the pairing known to the compiler and
// the encoding of infinite elements in a branch of its own: instructions, 2.8 a cycle and busy SM, against 13 for the bytes.
constexpr int WRITE_EACH = 4, WRITE_FILL = 148 * 4;
constexpr int WRITE_THREADS = 256;

// PAIRING 0: element i of the first half with element i of the second; 1: neighbours.  HD: the head size, or 0 where it is known at the launch only.
// Blocks an SM: of float32, whose items take twice the registers, 3 (4,096 rows of 28 + 4 + 4 heads: 30.5 us, with the bias asked for ahead 34, and
// 39 with four blocks).  The bias of bfloat16 is asked for ahead (prompts above: 25.7 us, else 28).
template <typename TA, typename TB, bool RUNS, int HD, int PAIRING>
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
    const int ia = PAIRING == 0 ? i : 2 * i, ib = PAIRING == 0 ? i + half : 2 * i + 8;       // where the item's two halves lie in the head
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
            for (int e = 0; e < 8; ++e) { lo.v[e] += x.v[e]; hi.v[e] += y.v[e]; }
        }
        if (RUNS && k + 1 < each) ask(j + side);                      // on its way while this one is worked on
        if (mine) {
            if (j < a.nh + c.nkv && a.cos_t != nullptr) {
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    if (PAIRING == 0) rotate(lo.v[e], hi.v[e], cs.v[e], sn.v[e]);
                    else rotate((e < 4 ? lo : hi).v[2 * (e & 3)], (e < 4 ? lo : hi).v[2 * (e & 3) + 1], cs.v[e], sn.v[e]);
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
            if (!infinite) {
                *reinterpret_cast<uint2*>(d + ia) = encode8<false>(lo, inv);
                *reinterpret_cast<uint2*>(d + ib) = encode8<false>(hi, inv);
            } else {
                *reinterpret_cast<uint2*>(d + ia) = encode8<true>(lo, inv);
                *reinterpret_cast<uint2*>(d + ib) = encode8<true>(hi, inv);
            }
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
TQ_EXPORT int tq_write8(const void* packed, int bytes) {
    C8_REQUIRE_CALL("write8", Write8Call);
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
    WriteArgs a{cos_t, sin_t, x.positions, x.cu_seqlens, x.held, nh, codes != nullptr ? nh + 2 * nkv : nh, 1};
    // a run of n rows touches at most (n + 14) / 16 + 1 blocks
    const bool runs = max_q_len > 1;
    const int units = runs ? (max_q_len + 14) / C8_BLOCK + 1 : 1, threads = runs ? (hd + 31) / 32 * 32 : 32;
    const int side = runs ? WRITE_THREADS / threads : n_seqs >= 32 ? 8 : 2;              // units a block takes side by side
    const long long blocks = (long long)units * ((a.written + side - 1) / side) * n_seqs;
    a.each = runs ? (int)max(1ll, min((long long)WRITE_EACH, blocks / WRITE_FILL)) : 1;
    const dim3 grid(units, (a.written + side * a.each - 1) / (side * a.each), n_seqs);
    TQ_DISPATCH(x.act_dtype, TA, TQ_DISPATCH(bias != nullptr ? x.bias_dtype : x.act_dtype, TB,
        const auto launch = [&](auto kernel) { tq_launch(grid, side * threads, 0, x.stream)(kernel, (const TA*)qkv, (const TB*)bias, a, (TA*)x.q_out, c, threads); };
        const auto of_pairing = [&](auto pairing) {
            constexpr int P = decltype(pairing)::value;
            if (runs) launch(hd == 128 ? write8_kernel<TA, TB, true, 128, P> : hd == 64 ? write8_kernel<TA, TB, true, 64, P> : write8_kernel<TA, TB, true, 0, P>);
            else launch(hd == 128 ? write8_kernel<TA, TB, false, 128, P> : write8_kernel<TA, TB, false, 0, P>);
        };
        if (x.pairing == 0) of_pairing(std::integral_constant<int, 0>()); else of_pairing(std::integral_constant<int, 1>())));
    TQ_CHECK_LAUNCH("write8");
    return 0;
}
