// Attention over the 8-bit cache (layout and codes: cache8.cuh) for single tokens, short runs and every type and head size.
//
//   tq_attention8   softmax(scale q.K) V, causal, with an optional window, the keys of a row cut into ranges that a second launch joins
//   tq_weigh8       sums of softmax weights: what each cached row received from a step's rows and its key/value head's query heads
//
// A CTA takes one key/value head of one sequence, a tile of 8 or 16 columns (query heads of one row, or of several rows of the run) and a range
// of the keys; its four warps take blocks of 16 keys in turn.  Both products run on mma.sync with the cache as the left operand, straight
// from global memory to registers: a lane's 16 bytes of a key row are its share of four steps of S = K q (which element goes to which place
// of a sum does not matter as long as the queries lie the same way), and its 16 bytes of four value rows, interleaved two rows at a time by
// byte permutes, its share of eight steps of O = V^T p.  No byte of the cache passes through shared memory.  Codes become float16 exactly
// (one conversion for two); so the queries are float16 as well, scaled per row by a power of two (bfloat16 ones are then exact down to
// 2^-24 of half the row's largest), float32 ones as two parts of 11 bits each.
//
// A block's two bytes are uniform over its 16 keys.  The key's scale goes into the factor that makes a sum a score.  The value's cannot go
// into float16 weights or values as it is (it spans 2^-126 .. 2^120), so the weights are taken as 2^(s + e - m'), m' the running maximum of s + e: at
// most 1, and what is lost below float16's range is lost against the largest contribution to the result.  The denominator has a
// maximum of its own, over s.
#include "cache8.cuh"

TQ_DEFINE_LAST_ERROR

namespace {

constexpr float LOG2E = 1.4426950408889634f;
constexpr int WARPS = 4;

__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
// D[16 x 8] += A[16 x 16] B[16 x 8], float16 operands
__device__ __forceinline__ void mma(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t transpose8x8(uint32_t x) {
    uint32_t y;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
    return y;
}
__device__ __forceinline__ uint32_t half2_of(float lo, float hi) {
    uint32_t d;
    asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(d) : "f"(hi), "f"(lo));
    return d;
}
__device__ __forceinline__ float2 float2_of(uint32_t h) {
    float2 f;
    asm("{\n\t.reg .b16 l, h;\n\tmov.b32 {l, h}, %2;\n\tcvt.f32.f16 %0, l;\n\tcvt.f32.f16 %1, h;\n\t}" : "=f"(f.x), "=f"(f.y) : "r"(h));
    return f;
}

struct Step {
    const int *cu_seqlens, *held;
    int nh, window;
    float factor;              // scale * log2(e)
};

// A tile of columns: query heads of one key/value head and rows of one run.
struct Tile {
    int t_begin, run, start, per, first, n;           // n columns from number `first` on, counted row by row
    int seq, g;
    __device__ __forceinline__ int row(int col) const { return (first + col) / per; }
    __device__ __forceinline__ size_t query(int col, const Step& S) const {           // row of q as [T * nh]
        const int c = first + col, r = c / per;
        return (size_t)(t_begin + r) * S.nh + g * per + (c - r * per);
    }
};
__device__ __forceinline__ Tile tile_of(const Step& S, int seq, int g, int nkv, int number, int columns) {
    Tile t;
    t.seq = seq; t.g = g;
    t.t_begin = S.cu_seqlens[seq];
    t.run = S.cu_seqlens[seq + 1] - t.t_begin;
    t.start = S.held[seq];
    t.per = S.nh / nkv;
    t.first = number * columns;
    t.n = min(columns, t.run * t.per - t.first);
    return t;
}

// The tile's queries in shared memory as right operands, [part][8 columns][step of 16 elements][lane], and each column's factor: score =
// (sum of the products) * factor * 2^(key byte - 127).
template <typename TA, int HDP, int NT> struct Queries {
    static constexpr int PARTS = sizeof(TA) == 4 ? 2 : 1, STEPS = HDP / 16;
    uint2 b[PARTS][NT][STEPS][32];
    float factor[NT * 8], up[NT * 8];
    __device__ void load(const TA* q, const Tile& t, const Step& S, int hd) {
        const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
        for (int c = warp; c < NT * 8; c += WARPS) {
            uint32_t top = 0;
            if (c < t.n) {
                const TA* row = q + t.query(c, S) * hd;
                for (int d = lane; d < hd; d += 32) top = max(top, c8_magnitude(tq_to_float(row[d])));
            }
            top = __reduce_max_sync(0xffffffffu, top);
            if (lane == 0) {
                // the largest element to between 2^14 and 2^15
                const int shift = min(126, 14 - max((int)(top >> 23) - 127, -126));
                up[c] = __uint_as_float((uint32_t)(127 + shift) << 23);
                factor[c] = S.factor * __uint_as_float((uint32_t)(127 - shift) << 23);
            }
        }
        __syncthreads();
        for (int i = threadIdx.x; i < NT * STEPS * 32; i += WARPS * 32) {
            const int l = i & 31, step = i / 32 % STEPS, nt = i / 32 / STEPS, c = nt * 8 + (l >> 2), d = (step / 4) * 64 + (l & 3) * 16 + (step & 3) * 4;
            float f[4] = {0.f, 0.f, 0.f, 0.f};
            if (c < t.n && d < hd) {
                const TA* row = q + t.query(c, S) * hd + d;
#pragma unroll
                for (int e = 0; e < 4; ++e) f[e] = tq_to_float(row[e]) * up[c];
            }
            const uint2 hi = make_uint2(half2_of(f[0], f[1]), half2_of(f[2], f[3]));
            b[0][nt][step][l] = hi;
            if (PARTS == 2) {
                const float2 x = float2_of(hi.x), y = float2_of(hi.y);
                // (what is not finite stays in the first part alone)
                auto left = [](float v, float h) { const float r = v - h; return fabsf(r) < INFINITY ? r : 0.f; };
                b[PARTS - 1][nt][step][l] = make_uint2(half2_of(left(f[0], x.x), left(f[1], x.y)), half2_of(left(f[2], y.x), left(f[3], y.y)));
            }
        }
        __syncthreads();
    }
};

// A lane's codes of a block of 16 keys: K rows lane / 4 and 8 more, 16 bytes of every 64; V rows 2 (lane % 4) and the next, and 8 more of both.
template <int HDP> struct KeyRegs { uint4 k[HDP / 64][2]; };
template <int HDP> struct ValueRegs { uint4 v[HDP > 128 ? 2 : 1][4]; };

template <int HDP>
__device__ __forceinline__ void load_keys(KeyRegs<HDP>& r, const uint8_t* rows, int hd) {
    const int lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
#pragma unroll
    for (int j = 0; j < HDP / 64; ++j) {
        const int d = j * 64 + t * 16;
#pragma unroll
        for (int h = 0; h < 2; ++h)
            r.k[j][h] = d < hd ? __ldg(reinterpret_cast<const uint4*>(rows + (size_t)(g + 8 * h) * hd + d)) : make_uint4(0, 0, 0, 0);
    }
}
template <int HDP>
__device__ __forceinline__ void load_values(ValueRegs<HDP>& r, const uint8_t* rows, int hd) {
    const int lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
#pragma unroll
    for (int j = 0; j < (HDP > 128 ? 2 : 1); ++j)
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            const int row = 2 * t + (k & 1) + 8 * (k >> 1);
            if (HDP == 64) {
                const uint2 x = g * 8 < hd ? __ldg(reinterpret_cast<const uint2*>(rows + (size_t)row * hd + g * 8)) : make_uint2(0, 0);
                r.v[j][k] = make_uint4(x.x, x.y, 0, 0);
            } else {
                const int d = j * 128 + g * 16;
                r.v[j][k] = d < hd ? __ldg(reinterpret_cast<const uint4*>(rows + (size_t)row * hd + d)) : make_uint4(0, 0, 0, 0);
            }
        }
}
__device__ __forceinline__ uint32_t word(const uint4& v, int i) { return i == 0 ? v.x : i == 1 ? v.y : i == 2 ? v.z : v.w; }

// Scores of a block: s[nt] = {key g column 2t, key g column 2t + 1, key g + 8 ..}, without their factors.
template <typename TA, int HDP, int NT>
__device__ __forceinline__ void products(float (&s)[NT][4], const KeyRegs<HDP>& r, const Queries<TA, HDP, NT>& Q) {
    const int lane = threadIdx.x & 31;
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) s[nt][0] = s[nt][1] = s[nt][2] = s[nt][3] = 0.f;
#pragma unroll
    for (int j = 0; j < HDP / 64; ++j)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const uint32_t x = word(r.k[j][0], i), y = word(r.k[j][1], i);
            const uint32_t a0 = c8_half2(x & 0xffffu), a2 = c8_half2(x >> 16), a1 = c8_half2(y & 0xffffu), a3 = c8_half2(y >> 16);
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                for (int p = 0; p < Queries<TA, HDP, NT>::PARTS; ++p) {
                    const uint2 b = Q.b[p][nt][j * 4 + i][lane];
                    mma(s[nt], a0, a1, a2, a3, b.x, b.y);
                }
        }
}

// Where a row of the step looks: the first and the last of its places.
__device__ __forceinline__ int first_seen(int place, int window) { return window > 0 ? max(0, place + 1 - window) : 0; }

// ---------------------------------------------------------------------------------------
// A range of the keys for a tile of columns.  partial: null, or [T * nh][ranges][hd + 4] for a second launch: the unnormalised sum, the
// maximum m' it is relative to, the denominator's maximum and the denominator.  scores: null, or [T * nh][score_stride], base-2 scores.
// lse: null, or [T * nh], log2 of the denominator (where there is no second launch).
// ---------------------------------------------------------------------------------------
template <typename TA, int HDP, int NT>
__device__ __forceinline__ void attend_tile(const Tile& T, int range, int ranges, const TA* __restrict__ q, const Cache8& c, const Step& S, TA* __restrict__ out,
                                            float* __restrict__ partial, float* __restrict__ scores, int score_stride, float* __restrict__ lse) {
    constexpr int NC = NT * 8, MT = HDP / 16;
    __shared__ Queries<TA, HDP, NT> Q;
    __shared__ float s_o[WARPS][NC][HDP + 4];
    __shared__ float s_stat[WARPS][NC][3];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3, hd = c.hd;
    // this range's blocks of 16 keys
    const int place0 = T.start + T.row(0), place1 = T.start + T.row(T.n - 1);
    const int block0 = first_seen(place0, S.window) / C8_BLOCK, blocks = place1 / C8_BLOCK + 1 - block0;
    const int each = (blocks + ranges * WARPS - 1) / (ranges * WARPS) * WARPS;
    const int from = block0 + range * each, to = min(from + each, block0 + blocks);
    Q.load(q, T, S, hd);

    int place_of[NT][2];               // the lane's columns' places (columns that are not there see nothing)
    float f[NT][2];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            const int col = nt * 8 + 2 * t + j;
            place_of[nt][j] = col < T.n ? T.start + T.row(col) : -1;
            f[nt][j] = Q.factor[col];
        }
    float o[NT][MT][4], m[NT][2], mo[NT][2], l[NT][2];        // m: of the scores, mo: of scores and value scales
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
        for (int i = 0; i < MT; ++i) o[nt][i][0] = o[nt][i][1] = o[nt][i][2] = o[nt][i][3] = 0.f;
        m[nt][0] = m[nt][1] = mo[nt][0] = mo[nt][1] = -INFINITY;
        l[nt][0] = l[nt][1] = 0.f;
    }
    KeyRegs<HDP> kr;
    ValueRegs<HDP> vr;
    uint32_t kb = 1, vb = 1;
    auto fetch = [&](int b, int page, KeyRegs<HDP>& k, ValueRegs<HDP>& v) {
        const int row = b * C8_BLOCK % c.page_size;
        load_keys<HDP>(k, c.codes + c.codes_at(page, 0, T.g) + (size_t)row * hd, hd);
        load_values<HDP>(v, c.codes + c.codes_at(page, 1, T.g) + (size_t)row * hd, hd);
        kb = c.scales[c.scales_at(page, 0, T.g) + row / C8_BLOCK];
        vb = c.scales[c.scales_at(page, 1, T.g) + row / C8_BLOCK];
    };
    int b = from + warp;
    if (b < to) fetch(b, c.page_of(T.seq, b * C8_BLOCK), kr, vr);
    int next_page = b + WARPS < to ? c.page_of(T.seq, (b + WARPS) * C8_BLOCK) : 0;
    for (; b < to; b += WARPS) {
        const KeyRegs<HDP> kc = kr;
        const ValueRegs<HDP> vc = vr;
        const float ks = c8_scale(kb), ve = (float)((int)vb - 127);
        if (b + WARPS < to) {
            fetch(b + WARPS, next_page, kr, vr);
            next_page = b + 2 * WARPS < to ? c.page_of(T.seq, (b + 2 * WARPS) * C8_BLOCK) : 0;
        }
        float s[NT][4];
        products<TA, HDP, NT>(s, kc, Q);
        const int key = b * C8_BLOCK + g;
        // every column sees all 16 keys? (those that are not there may see them too: nobody reads their sums)
        const bool whole = b * C8_BLOCK + C8_BLOCK - 1 <= place0 && (S.window <= 0 || b * C8_BLOCK > place1 - S.window);
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                s[nt][j] = s[nt][j] * (f[nt][j & 1] * ks);
                const int p = place_of[nt][j & 1], k = key + 8 * (j >> 1);
                if (!whole && (k > p || (S.window > 0 && k <= p - S.window))) s[nt][j] = -INFINITY;
            }
        if (scores != nullptr) {
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const int col = nt * 8 + 2 * t + (j & 1);
                    if (col < T.n && key + 8 * (j >> 1) < score_stride) scores[T.query(col, S) * score_stride + key + 8 * (j >> 1)] = s[nt][j];
                }
        }
        // the maxima grow now and then: found by all lanes of a column together when one of them sees a larger value
        bool grows = false;
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int j = 0; j < 4; ++j) grows |= s[nt][j] > m[nt][j & 1] || s[nt][j] + ve > mo[nt][j & 1];
        if (__any_sync(0xffffffffu, grows)) {
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                for (int j = 0; j < 2; ++j) {
                    float top = fmaxf(s[nt][j], s[nt][j + 2]);
#pragma unroll
                    for (int x = 4; x < 32; x <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, x));
                    const float mn = fmaxf(m[nt][j], top), mon = fmaxf(mo[nt][j], top + ve);
                    if (mn > m[nt][j]) { l[nt][j] *= ex2(m[nt][j] - mn); m[nt][j] = mn; }
                    if (mon > mo[nt][j]) {
                        const float down = ex2(mo[nt][j] - mon);
#pragma unroll
                        for (int i = 0; i < MT; ++i) { o[nt][i][j] *= down; o[nt][i][j + 2] *= down; }
                        mo[nt][j] = mon;
                    }
                }
        }
        uint32_t p_hi[NT][2], p_lo[NT][2];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
            float w[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const float mr = m[nt][j & 1] == -INFINITY ? 0.f : m[nt][j & 1], mor = mo[nt][j & 1] == -INFINITY ? 0.f : mo[nt][j & 1];
                l[nt][j & 1] += ex2(s[nt][j] - mr);
                w[j] = ex2(s[nt][j] + ve - mor);
            }
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const uint32_t hi = half2_of(w[2 * h], w[2 * h + 1]);
                p_hi[nt][h] = transpose8x8(hi);
                if (Queries<TA, HDP, NT>::PARTS == 2) {
                    const float2 x = float2_of(hi);
                    p_lo[nt][h] = transpose8x8(half2_of(w[2 * h] - x.x, w[2 * h + 1] - x.y));
                }
            }
        }
        // Values no column may see come with a weight of 0, which does not remove a NaN: such codes are taken out of the product, and put
        // back as NaN into the sums of the columns that do see the key.
        ValueRegs<HDP> vm = vc;
        uint32_t lost[HDP > 128 ? 2 : 1][4] = {};             // of the lane's four rows: which of its 16 elements are NaN
        bool some = false;
        if (!whole) {
#pragma unroll
            for (int j = 0; j < (HDP > 128 ? 2 : 1); ++j)
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    uint32_t* u = &vm.v[j][k].x;
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const uint32_t hit = ((u[i] & 0x7f7f7f7fu) + 0x01010101u) & 0x80808080u;     // the top bit of every byte 0x7f or 0xff
                        lost[j][k] |= ((hit >> 7 & 1u) | (hit >> 14 & 2u) | (hit >> 21 & 4u) | (hit >> 28 & 8u)) << (4 * i);
                        u[i] &= ~((hit >> 7) * 0xffu);
                    }
                    some |= lost[j][k] != 0;
                }
            some = __any_sync(0xffffffffu, some);
        }
#pragma unroll
        for (int i = 0; i < MT; i += 2) {
            // words i / 2 of the lane's four rows: two steps of 16 elements
            const int j = HDP > 128 ? i / 8 : 0, wd = (i - 8 * j) / 2;
            const uint32_t r0 = word(vm.v[j][0], wd), r1 = word(vm.v[j][1], wd), r2 = word(vm.v[j][2], wd), r3 = word(vm.v[j][3], wd);
            const uint32_t x = __byte_perm(r0, r1, 0x5140), y = __byte_perm(r0, r1, 0x7362), z = __byte_perm(r2, r3, 0x5140), v = __byte_perm(r2, r3, 0x7362);
            const uint32_t a0 = c8_half2(x & 0xffffu), a1 = c8_half2(x >> 16), a2 = c8_half2(z & 0xffffu), a3 = c8_half2(z >> 16);
            const uint32_t e0 = c8_half2(y & 0xffffu), e1 = c8_half2(y >> 16), e2 = c8_half2(v & 0xffffu), e3 = c8_half2(v >> 16);
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
                mma(o[nt][i], a0, a1, a2, a3, p_hi[nt][0], p_hi[nt][1]);
                mma(o[nt][i + 1], e0, e1, e2, e3, p_hi[nt][0], p_hi[nt][1]);
                if (Queries<TA, HDP, NT>::PARTS == 2) {
                    mma(o[nt][i], a0, a1, a2, a3, p_lo[nt][0], p_lo[nt][1]);
                    mma(o[nt][i + 1], e0, e1, e2, e3, p_lo[nt][0], p_lo[nt][1]);
                }
            }
        }
        if (some) {
#pragma unroll 1
            for (int k16 = 0; k16 < C8_BLOCK; ++k16) {
                const int owner = (lane & ~3) | ((k16 & 7) >> 1), slot = (k16 & 1) + 2 * (k16 >> 3);
#pragma unroll
                for (int j = 0; j < (HDP > 128 ? 2 : 1); ++j) {
                    const uint32_t mine = slot == 0 ? lost[j][0] : slot == 1 ? lost[j][1] : slot == 2 ? lost[j][2] : lost[j][3];
                    const uint32_t bits = __shfl_sync(0xffffffffu, mine, owner);
                    const int k = b * C8_BLOCK + k16;
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                        for (int col = 0; col < 2; ++col) {
                            const int p = place_of[nt][col];
                            if (k > p || (S.window > 0 && k <= p - S.window)) continue;
#pragma unroll
                            for (int i = 0; i < (MT < 8 ? MT : 8); ++i) {
                                if (bits >> (2 * i) & 1u) o[nt][j * 8 + i][col] = NAN;
                                if (bits >> (2 * i + 1) & 1u) o[nt][j * 8 + i][col + 2] = NAN;
                            }
                        }
                }
            }
        }
    }
    // the warps' sums together
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int j = 0; j < 2; ++j) {
#pragma unroll
            for (int x = 4; x < 32; x <<= 1) l[nt][j] += __shfl_xor_sync(0xffffffffu, l[nt][j], x);
            const int col = nt * 8 + 2 * t + j;
            if (g == 0) { s_stat[warp][col][0] = mo[nt][j]; s_stat[warp][col][1] = m[nt][j]; s_stat[warp][col][2] = l[nt][j]; }
#pragma unroll
            for (int i = 0; i < MT; ++i) {
                const int d = HDP == 64 ? g * 8 + 2 * i : (i / 8) * 128 + g * 16 + 2 * (i % 8);
                *reinterpret_cast<float2*>(&s_o[warp][col][d]) = make_float2(o[nt][i][j], o[nt][i][j + 2]);
            }
        }
    __syncthreads();
    for (int col = warp; col < T.n; col += WARPS) {
        float mw[WARPS], M = -INFINITY, MO = -INFINITY, L = 0.f;
#pragma unroll
        for (int w = 0; w < WARPS; ++w) { MO = fmaxf(MO, s_stat[w][col][0]); M = fmaxf(M, s_stat[w][col][1]); }
#pragma unroll
        for (int w = 0; w < WARPS; ++w) {
            mw[w] = s_stat[w][col][0] == -INFINITY ? 0.f : exp2f(s_stat[w][col][0] - MO);
            // (a NaN in the denominator has to stay one)
            L += s_stat[w][col][1] == -INFINITY ? s_stat[w][col][2] : s_stat[w][col][2] * exp2f(s_stat[w][col][1] - M);
        }
        const size_t at = T.query(col, S);
        float* pp = partial != nullptr ? partial + (at * ranges + range) * (hd + 4) : nullptr;
        const float norm = exp2f(MO - M) / L;
        for (int d = lane; d < hd; d += 32) {
            float sum = 0.f;
#pragma unroll
            for (int w = 0; w < WARPS; ++w) sum += s_o[w][col][d] * mw[w];
            if (pp != nullptr) pp[d] = sum;
            else out[at * hd + d] = tq_from_float<TA>(sum * norm);
        }
        if (pp != nullptr && lane == 0) { pp[hd] = MO; pp[hd + 1] = M; pp[hd + 2] = L; }
        if (pp == nullptr && lse != nullptr && lane == 0) lse[at] = M + log2f(L);
    }
}

template <typename TA, int HDP, int NT>
__global__ void __launch_bounds__(WARPS * 32) attention8_kernel(const TA* __restrict__ q, Cache8 c, Step S, TA* __restrict__ out, float* __restrict__ partial,
                                                                float* __restrict__ scores, int score_stride, float* __restrict__ lse) {
    tq_grid_wait();                    // everything below may read what the previous kernel wrote
    tq_grid_launch_dependents();
    const int tile_no = blockIdx.x / c.nkv;
    const Tile T = tile_of(S, blockIdx.z, blockIdx.x - tile_no * c.nkv, c.nkv, tile_no, NT * 8);
    if (T.n > 0) attend_tile<TA, HDP, NT>(T, blockIdx.y, gridDim.y, q, c, S, out, partial, scores, score_stride, lse);
}

// The prompt kernel gives values that a row may not see a weight of 0, which does not remove a NaN: key/value heads of sequences in whose pages
// `lost` [n_seqs][nkv][pages] marks such values are done again here, all others cost a look at their marks.
template <typename TA, int HDP, int NT>
__global__ void __launch_bounds__(WARPS * 32) repair8_kernel(const TA* __restrict__ q, Cache8 c, Step S, TA* __restrict__ out, const uint8_t* __restrict__ lost,
                                                             int lost_stride, int page_size) {
    tq_grid_wait();                    // everything below may read what the previous kernel wrote
    tq_grid_launch_dependents();
    const int seq = blockIdx.z, g = blockIdx.y, start = S.held[seq], run = S.cu_seqlens[seq + 1] - S.cu_seqlens[seq];
    if (run <= 0) return;
    const uint8_t* marks = lost + ((size_t)seq * c.nkv + g) * lost_stride;
    bool some = false;
    for (int p = first_seen(start, S.window) / page_size + (int)threadIdx.x; p <= (start + run - 1) / page_size; p += WARPS * 32) some |= marks[p] != 0;
    if (!__syncthreads_or(some)) return;
    for (int tile_no = blockIdx.x; ; tile_no += gridDim.x) {
        const Tile T = tile_of(S, seq, g, c.nkv, tile_no, NT * 8);
        if (T.n <= 0) return;
        __syncthreads();
        attend_tile<TA, HDP, NT>(T, 0, 1, q, c, S, out, nullptr, nullptr, 0, nullptr);
    }
}

// ---------------------------------------------------------------------------------------
// The ranges of a row joined: block x = 0 of a (sequence, key/value head).  Further blocks add the row weights up from the scores the first
// launch left, 128 places each.
// ---------------------------------------------------------------------------------------
template <typename TA>
__global__ void __launch_bounds__(128) join8_kernel(Cache8 c, Step S, const float* __restrict__ partial, int ranges, TA* __restrict__ out,
                                                    float* __restrict__ lse, const float* __restrict__ scores, int score_stride, float* __restrict__ weights) {
    tq_grid_wait();                    // everything below may read what the previous kernel wrote
    tq_grid_launch_dependents();
    const int seq = blockIdx.z, g = blockIdx.y, per = S.nh / c.nkv, hd = c.hd, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int t_begin = S.cu_seqlens[seq], run = S.cu_seqlens[seq + 1] - t_begin, start = S.held[seq];
    if (run <= 0) return;
    // the statistics of a row over its ranges
    auto stats = [&](size_t at, float& MO, float& M, float& L) {
        const float* p = partial + at * ranges * (hd + 4) + hd;
        MO = -INFINITY; M = -INFINITY; L = 0.f;
        for (int r = lane; r < ranges; r += 32) { MO = fmaxf(MO, p[(size_t)r * (hd + 4)]); M = fmaxf(M, p[(size_t)r * (hd + 4) + 1]); }
        MO = tq_warp_max(MO);
        M = tq_warp_max(M);
        for (int r = lane; r < ranges; r += 32) {
            const float mr = p[(size_t)r * (hd + 4) + 1], lr = p[(size_t)r * (hd + 4) + 2];
            L += mr == -INFINITY ? lr : lr * exp2f(mr - M);
        }
        L = tq_warp_sum(L);
    };
    if (blockIdx.x == 0) {
        for (int c0 = warp; c0 < run * per; c0 += 4) {
            const int r0 = c0 / per;
            const size_t at = (size_t)(t_begin + r0) * S.nh + g * per + (c0 - r0 * per);
            float MO, M, L;
            stats(at, MO, M, L);
            const float norm = exp2f(MO - M) / L;
            if (lse != nullptr && lane == 0) lse[at] = M + log2f(L);
            const float* p = partial + at * ranges * (hd + 4);
            for (int d = lane; d < hd; d += 32) {
                float sum = 0.f;
                for (int r = 0; r < ranges; ++r) {
                    const float mr = p[(size_t)r * (hd + 4) + hd], v = p[(size_t)r * (hd + 4) + d];
                    sum += mr == -INFINITY ? v : v * exp2f(mr - MO);
                }
                out[at * hd + d] = tq_from_float<TA>(sum * norm);
            }
        }
        return;
    }
    __shared__ float s_lse[128];
    const int place = (blockIdx.x - 1) * 128 + threadIdx.x, columns = run * per;
    if ((int)(blockIdx.x - 1) * 128 >= start + run) return;
    float sum = 0.f;
    for (int c0 = 0; c0 < columns; c0 += 128) {
        __syncthreads();
        for (int x = warp; x < min(128, columns - c0); x += 4) {
            const int r0 = (c0 + x) / per;
            float MO, M, L;
            stats((size_t)(t_begin + r0) * S.nh + g * per + (c0 + x - r0 * per), MO, M, L);
            if (lane == 0) s_lse[x] = M + log2f(L);
        }
        __syncthreads();
        for (int x = 0; x < min(128, columns - c0); ++x) {
            const int r0 = (c0 + x) / per, p = start + r0;
            if (place > p || place >= score_stride || (S.window > 0 && place <= p - S.window)) continue;
            sum += ex2(scores[((size_t)(t_begin + r0) * S.nh + g * per + (c0 + x - r0 * per)) * score_stride + place] - s_lse[x]);
        }
    }
    if (place >= start + run || (S.window > 0 && place + S.window <= start)) return;       // no row of the step sees it
    float* w = weights + ((size_t)c.page_of(seq, place) * c.nkv + g) * c.page_size + place % c.page_size;
    *w = (place < start ? *w : 0.f) + sum;
}

// ---------------------------------------------------------------------------------------
// Sums of weights from the queries and the keys again: a warp keeps a block of 16 keys in registers and walks the columns that see it, 8
// or 16 at a time.  One writer per sum and a fixed order: the same bits every time.
// ---------------------------------------------------------------------------------------
template <typename TA, int HDP, int NT>
__global__ void __launch_bounds__(WARPS * 32) weigh8_kernel(const TA* __restrict__ q, Cache8 c, Step S, const float* __restrict__ lse, float* __restrict__ weights) {
    tq_grid_wait();                    // everything below may read what the previous kernel wrote
    tq_grid_launch_dependents();
    constexpr int NC = NT * 8;
    __shared__ Queries<TA, HDP, NT> Q;
    const int seq = blockIdx.z, gh = blockIdx.y, warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3, hd = c.hd;
    Tile T = tile_of(S, seq, gh, c.nkv, 0, NC);
    const int key0 = blockIdx.x * WARPS * C8_BLOCK, last_key = key0 + WARPS * C8_BLOCK - 1;
    // rows of the run that see some of the CTA's keys
    const int row0 = max(0, key0 - T.start), row1 = S.window > 0 ? min(T.run, last_key + S.window - T.start) : T.run;
    if (row0 >= row1) return;
    const int block = blockIdx.x * WARPS + warp, key = block * C8_BLOCK + g;
    const bool mine = block * C8_BLOCK < T.start + T.run && !(S.window > 0 && block * C8_BLOCK + C8_BLOCK - 1 + S.window <= T.start);
    KeyRegs<HDP> kr = {};
    float ks = 0.f;
    int page = 0;
    const int row = block * C8_BLOCK % c.page_size;
    if (mine) {
        page = c.page_of(seq, block * C8_BLOCK);
        load_keys<HDP>(kr, c.codes + c.codes_at(page, 0, gh) + (size_t)row * hd, hd);
        ks = c8_scale(c.scales[c.scales_at(page, 0, gh) + row / C8_BLOCK]);
    }
    float sum[2] = {0.f, 0.f};
    const int all = row1 * T.per;
    for (T.first = row0 * T.per; T.first < all; T.first += NC) {
        T.n = min(NC, all - T.first);
        __syncthreads();
        Q.load(q, T, S, hd);
        if (!mine) continue;
        float s[NT][4];
        products<TA, HDP, NT>(s, kr, Q);
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                const int col = nt * 8 + 2 * t + j;
                if (col >= T.n) continue;
                const int p = T.start + T.row(col);
                const float f = Q.factor[col] * ks, L = lse[T.query(col, S)];
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    const int k = key + 8 * h;
                    if (k <= p && (S.window <= 0 || k > p - S.window)) sum[h] += ex2(s[nt][j + 2 * h] * f - L);
                }
            }
    }
    if (!mine) return;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        sum[h] += __shfl_xor_sync(0xffffffffu, sum[h], 1);
        sum[h] += __shfl_xor_sync(0xffffffffu, sum[h], 2);
        const int k = key + 8 * h;
        if (t == 0 && k < T.start + T.run && !(S.window > 0 && k + S.window <= T.start)) {
            float* w = weights + ((size_t)page * c.nkv + gh) * c.page_size + row + g + 8 * h;
            *w = (k < T.start ? *w : 0.f) + sum[h];
        }
    }
}

template <typename TA, int HDP, int NT>
int launch8(const void* q, const Cache8& c, const Step& S, void* out, float* partial, int ranges, float* scores, int score_stride, float* lse, int n_seqs,
            int max_q_len, cudaStream_t stream) {
    const long long tiles = ((long long)max_q_len * (S.nh / c.nkv) + NT * 8 - 1) / (NT * 8) * c.nkv;
    TQ_REQUIRE(tiles < (1ll << 31), "attention8: runs of %d rows", max_q_len);
    tq_launch(dim3((unsigned)tiles, ranges, n_seqs), WARPS * 32, 0, stream)(attention8_kernel<TA, HDP, NT>, (const TA*)q, c, S, (TA*)out, partial, scores, score_stride, lse);
    TQ_CHECK_LAUNCH("attention8");
    return 0;
}
template <typename TA, int HDP, int NT>
int launch_weigh8(const void* q, const Cache8& c, const Step& S, const float* lse, float* weights, int n_seqs, int max_kv_len, cudaStream_t stream) {
    const int per_cta = WARPS * C8_BLOCK;
    tq_launch(dim3((max_kv_len + per_cta - 1) / per_cta, c.nkv, n_seqs), WARPS * 32, 0, stream)(weigh8_kernel<TA, HDP, NT>, (const TA*)q, c, S, lse, weights);
    TQ_CHECK_LAUNCH("weigh8");
    return 0;
}
// Two tiles of 8 columns where there are more than 8 (heads of up to 128: beyond, the sums of 16 columns do not fit the registers)
#define C8_SIZES(columns, CALL)                                                                          \
    do {                                                                                                 \
        if (hd <= 64) { if ((columns) > 8) return CALL(64, 2); return CALL(64, 1); }                     \
        if (hd <= 128) { if ((columns) > 8) return CALL(128, 2); return CALL(128, 1); }                  \
        return CALL(256, 1);                                                                             \
    } while (0)

int check_step(const char* what, int nh, int nkv, int n_seqs, int longest, int window) {
    TQ_REQUIRE(nh >= 1 && nh % nkv == 0 && nkv <= 65535, "%s: %d heads are not a multiple of %d key/value heads", what, nh, nkv);
    TQ_REQUIRE(n_seqs <= 65535 && longest >= 1 && window >= 0, "%s: %d sequences, longest %d, window %d", what, n_seqs, longest, window);
    return 0;
}

}  // namespace

// q [T, nh, hd], out [T, nh * hd]; place i sees j <= i with window == 0 or i - j < window.  max_q_len: the longest run.  ranges > 1: the keys
// of a row are cut into that many ranges, partial [T * nh * ranges * (hd + 4)].  lse [T, nh] float32 or null.  scores [T * nh,
// score_stride] with weights [n_pages, nkv, page_size], or both null: the weights are added up by the second launch (any number of ranges
// needs partial then); score_stride: a multiple of 16, at least the longest held[s] + run, max_kv_len.
TQ_EXPORT int tq_attention8(const void* q, const void* codes, const void* scales, int act_dtype, const int* cu_seqlens, const int* held,
                            const int* page_table, int table_stride, int page_size, int window, float scale, void* out, float* partial, int ranges,
                            float* lse, float* scores, int score_stride, float* weights, int max_kv_len, int n_pages, int n_seqs, int max_q_len, int nh,
                            int nkv, int hd, cudaStream_t stream) {
    if (n_seqs == 0 || max_q_len == 0) return 0;
    int rc = c8_check("attention8", codes, scales, page_size, n_pages, nkv, hd, table_stride);
    if (!rc) rc = check_step("attention8", nh, nkv, n_seqs, max_q_len, window);
    if (rc) return rc;
    TQ_REQUIRE(ranges >= 1 && ranges <= 65535 && (ranges == 1 || partial != nullptr), "attention8: %d ranges need a buffer for their sums", ranges);
    TQ_REQUIRE((scores == nullptr) == (weights == nullptr) && (scores == nullptr || (partial != nullptr && score_stride % 16 == 0 && score_stride >= max_kv_len)),
               "attention8: scores of %d places do not hold %d", score_stride, max_kv_len);
    const Cache8 c{(uint8_t*)codes, (uint8_t*)scales, page_table, table_stride, page_size, n_pages, nkv, hd};
    const Step S{cu_seqlens, held, nh, window, scale * LOG2E};
    const int columns = max_q_len * (nh / nkv);
    auto first = [&]() -> int {
        TQ_DISPATCH(act_dtype, TA,
#define C8_CALL(HDP, NT) (launch8<TA, HDP, NT>(q, c, S, out, partial, ranges, scores, score_stride, partial == nullptr ? lse : nullptr, n_seqs, max_q_len, stream))
            C8_SIZES(columns, C8_CALL));
#undef C8_CALL
        return -2;
    };
    rc = first();
    if (rc || partial == nullptr) return rc;
    const int chunks = weights != nullptr ? (max_kv_len + 127) / 128 : 0;
    TQ_DISPATCH(act_dtype, TA, tq_launch(dim3(1 + chunks, nkv, n_seqs), 128, 0, stream)(join8_kernel<TA>, c, S, partial, ranges, (TA*)out, lse, scores, score_stride, weights));
    TQ_CHECK_LAUNCH("join8");
    return 0;
}

// After a prompt kernel's launch over the same step (bfloat16, heads of 64 or 128): lost [n_seqs][nkv][lost_stride] marks the pages, counted
// within a sequence, that hold a NaN among the values the step sees.
TQ_EXPORT int tq_repair8(const void* q, const void* codes, const void* scales, const int* cu_seqlens, const int* held, const int* page_table, int table_stride,
                         int page_size, int window, float scale, void* out, const void* lost, int lost_stride, int n_pages, int n_seqs, int nh, int nkv, int hd,
                         cudaStream_t stream) {
    if (n_seqs == 0) return 0;
    int rc = c8_check("repair8", codes, scales, page_size, n_pages, nkv, hd, table_stride);
    if (!rc) rc = check_step("repair8", nh, nkv, n_seqs, 1, window);
    if (rc) return rc;
    TQ_REQUIRE(hd == 64 || hd == 128, "repair8: head size %d", hd);
    const Cache8 c{(uint8_t*)codes, (uint8_t*)scales, page_table, table_stride, page_size, n_pages, nkv, hd};
    const Step S{cu_seqlens, held, nh, window, scale * LOG2E};
    const int heads = nkv * n_seqs, each = heads >= 444 ? 1 : 444 / heads;
    using TA = __nv_bfloat16;
    if (hd == 64) tq_launch(dim3(each, nkv, n_seqs), WARPS * 32, 0, stream)(repair8_kernel<TA, 64, 2>, (const TA*)q, c, S, (TA*)out, (const uint8_t*)lost, lost_stride, page_size);
    else tq_launch(dim3(each, nkv, n_seqs), WARPS * 32, 0, stream)(repair8_kernel<TA, 128, 2>, (const TA*)q, c, S, (TA*)out, (const uint8_t*)lost, lost_stride, page_size);
    TQ_CHECK_LAUNCH("repair8");
    return 0;
}

// weights of places below held[s] grow by, those of the step's own rows become, the sum over the step's rows and the head's query heads of
// 2^(score - lse).  max_kv_len: at least the longest held[s] + run.
TQ_EXPORT int tq_weigh8(const void* q, const void* codes, const void* scales, int act_dtype, const int* cu_seqlens, const int* held,
                        const int* page_table, int table_stride, int page_size, int window, float scale, const float* lse, float* weights, int n_pages,
                        int n_seqs, int max_q_len, int max_kv_len, int nh, int nkv, int hd, cudaStream_t stream) {
    if (n_seqs == 0 || max_kv_len == 0) return 0;
    int rc = c8_check("weigh8", codes, scales, page_size, n_pages, nkv, hd, table_stride);
    if (!rc) rc = check_step("weigh8", nh, nkv, n_seqs, max_kv_len, window);
    if (rc) return rc;
    const Cache8 c{(uint8_t*)codes, (uint8_t*)scales, page_table, table_stride, page_size, n_pages, nkv, hd};
    const Step S{cu_seqlens, held, nh, window, scale * LOG2E};
    const int columns = max_q_len * (nh / nkv);
    TQ_DISPATCH(act_dtype, TA,
#define C8_CALL(HDP, NT) (launch_weigh8<TA, HDP, NT>(q, c, S, lse, weights, n_seqs, max_kv_len, stream))
        C8_SIZES(columns, C8_CALL));
#undef C8_CALL
    return -2;
}
