// Attention over the 8-bit cache (layout and codes: cache8.cuh) for single tokens, short runs and every type and head size.
//
//   tq_attention8   softmax(scale q.K) V, causal, with an optional window, the keys of a row cut into ranges: up to 8 join as a cluster, more in a
//                   second launch
//   tq_weigh8       sums of softmax weights: what each cached row received from a step's rows and its key/value head's query heads
//
// A CTA takes one key/value head of one sequence, a tile of 8 or 16 columns (query heads of one row, or of several rows of the run) and a range
// of the keys; its four warps take blocks of 16 keys in turn, each through a ring of its own in shared memory that cp.async fills two blocks ahead (in
// tq_weigh8 keys go straight to registers).  Both products run on mma.sync with the cache as the left operand: a lane's 16 bytes of a key row are its
// share of four steps of S = K q (which element goes to which place of a sum does not matter as long as the queries lie the same way), and its
// 16 bytes of four value rows, interleaved two rows at a time by byte permutes, its share of eight steps of O = V^T p.  Codes become float16
// exactly (one conversion for two); so the queries are float16 as well, scaled per row by a power of two (bfloat16 ones are then exact down to
// 2^-24 of half the row's largest), float32 ones as two parts of 11 bits each.
//
// A block's two bytes are uniform over its 16 keys.  The key's scale goes into the factor that makes a sum a score.  The value's cannot go
// into float16 weights or values as it is (it spans 2^-126 .. 2^120), so the weights are taken as 2^(s + e - m'), m' the running maximum of s + e, times
// 2^14: at most 2^14, so that float16 holds them to 11 bits down to 2^-28 of the largest and to multiples of 2^-38 of it (without the
// factor down to 2^-14 and 2^-24: thousands of keys beside one that most of the weight goes to, 2^-22 of it each, then lose a hundredth of their sum).
// What is lost below that is lost against the largest contribution to the row's result, over all of its elements: an element that is zero in a
// block whose byte is 30 above the others' has some eight bits of those.  The denominator has a maximum of its own, over s.  m' is kept as its
// distance from that one: differences of scores are exact where they matter, sums of a score and an exponent are not once scores are large.
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
constexpr int CLUSTER = 8;     // ranges of a row that join through one another's shared memory

// A tile of columns: query heads of one key/value head and rows of one run.
struct Tile {
    int t_begin, run, start, per, first, n;           // n columns from number `first` on, counted row by row
    int seq, g;
    __device__ __forceinline__ int row(int col) const { return per == 1 ? first + col : (first + col) / per; }
    __device__ __forceinline__ size_t query(int col, const Step& S) const {           // row of q as [T * nh]
        const int c = first + col, r = row(col);
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

// Head sizes: HDP elements have registers; EXACT: the head has just that many (its offsets are then constants), else a multiple of 16 below.
template <typename TA_, int HDP_, int NT_, bool EXACT_> struct Form {
    using TA = TA_;
    static constexpr int HDP = HDP_, NT = NT_, NC = NT * 8, MT = HDP / 16, STEPS = HDP / 16, PARTS = sizeof(TA) == 4 ? 2 : 1;
    static constexpr bool EXACT = EXACT_, KEEP = NT * PARTS == 1 && HDP <= 128;       // KEEP: the queries stay in registers
    static constexpr int VG = HDP > 128 ? 2 : 1, STAGES = 3, STAGE_BYTES = 2 * C8_BLOCK * HDP, RING = WARPS * STAGES * STAGE_BYTES, SUMS = WARPS * NC * (HDP + 4) * 4;
    static constexpr int SMEM = RING > SUMS ? RING : SUMS;
    static constexpr int PER_SM = HDP > 128 ? 2 : HDP * NT > 128 ? 3 : 4;              // CTAs an SM holds (the registers' limit)
};

// Which 16 elements of a key row a lane's piece j is: a quarter of the lanes (t = lane % 4) holds each, two by two so that even and odd rows meet in
// no bank (see Piece).
template <int HDP> __device__ __forceinline__ int chunk_of(int j, int t) { return HDP == 64 ? t : 2 * t + (j & 1) + 8 * (j >> 1); }

// Four elements of a row, whose offset is a multiple of four elements (B200, element by element: 64 single steps of 16 heads of 128 84 us, now
// 80; 678 rows of 28 heads of 128 in float32 71 us, now 58).
__device__ __forceinline__ void load4(float (&x)[4], const __nv_bfloat16* p, bool aligned) {
    if (aligned) {
        const uint2 v = *reinterpret_cast<const uint2*>(p);
        x[0] = __uint_as_float(v.x << 16); x[1] = __uint_as_float(v.x & 0xffff0000u);
        x[2] = __uint_as_float(v.y << 16); x[3] = __uint_as_float(v.y & 0xffff0000u);
    } else {
#pragma unroll
        for (int e = 0; e < 4; ++e) x[e] = tq_to_float(p[e]);
    }
}
__device__ __forceinline__ void load4(float (&x)[4], const float* p, bool aligned) {
    if (aligned) {
        const float4 v = *reinterpret_cast<const float4*>(p);
        x[0] = v.x; x[1] = v.y; x[2] = v.z; x[3] = v.w;
    } else {
#pragma unroll
        for (int e = 0; e < 4; ++e) x[e] = p[e];
    }
}

// The tile's queries in shared memory as right operands, [part][8 columns][step of 16 elements][lane], each column's factor (score =
// (sum of the products) * factor * 2^(key byte - 127)), its row in q and its place (columns that are not there: place -1).
template <class F> struct Queries {
    uint2 b[F::PARTS][F::NT][F::STEPS][32];
    float factor[F::NC], up[F::NC];
    int place[F::NC];
    size_t row[F::NC];
    __device__ __forceinline__ void load(const typename F::TA* q, const Tile& t, const Step& S, int hd) {
        const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
        const bool aligned = ((uintptr_t)q & 15) == 0;
        constexpr int OWN = F::NC / WARPS, EACH = (F::HDP + 127) / 128;       // columns a warp looks over, pieces of four elements a lane
        float x[OWN][EACH][4];                 // all asked for before the first is used
        size_t rows[OWN];
#pragma unroll
        for (int o = 0; o < OWN; ++o) {
            const int c = warp + o * WARPS;
            rows[o] = c < t.n ? t.query(c, S) : 0;
#pragma unroll
            for (int k = 0; k < EACH; ++k) {
                x[o][k][0] = x[o][k][1] = x[o][k][2] = x[o][k][3] = 0.f;
                if (c < t.n && (lane + 32 * k) * 4 < hd) load4(x[o][k], q + rows[o] * hd + (lane + 32 * k) * 4, aligned);
            }
        }
#pragma unroll
        for (int o = 0; o < OWN; ++o) {
            const int c = warp + o * WARPS;
            const size_t at = rows[o];
            uint32_t top = 0;
#pragma unroll
            for (int k = 0; k < EACH; ++k)
#pragma unroll
                for (int e = 0; e < 4; ++e) top = max(top, c8_magnitude(x[o][k][e]));
            top = __reduce_max_sync(0xffffffffu, top);
            if (lane == 0) {
                // the largest element to between 2^14 and 2^15
                const int shift = min(126, 14 - max((int)(top >> 23) - 127, -126));
                up[c] = __uint_as_float((uint32_t)(127 + shift) << 23);
                factor[c] = S.factor * __uint_as_float((uint32_t)(127 - shift) << 23);
                place[c] = c < t.n ? t.start + t.row(c) : -1;
                row[c] = at;
            }
        }
        __syncthreads();
        for (int i = threadIdx.x; i < F::NT * F::STEPS * 32; i += WARPS * 32) {
            const int l = i & 31, step = i / 32 % F::STEPS, nt = i / 32 / F::STEPS, c = nt * 8 + (l >> 2), d = chunk_of<F::HDP>(step / 4, l & 3) * 16 + (step & 3) * 4;
            float f[4] = {0.f, 0.f, 0.f, 0.f};
            if (c < t.n && d < hd) {
                load4(f, q + row[c] * hd + d, aligned);
#pragma unroll
                for (int e = 0; e < 4; ++e) f[e] *= up[c];
            }
            const uint2 hi = make_uint2(half2_of(f[0], f[1]), half2_of(f[2], f[3]));
            b[0][nt][step][l] = hi;
            if (F::PARTS == 2) {
                const float2 x = float2_of(hi.x), y = float2_of(hi.y);
                // (what is not finite stays in the first part alone)
                auto left = [](float v, float h) { const float r = v - h; return fabsf(r) < INFINITY ? r : 0.f; };
                b[F::PARTS - 1][nt][step][l] = make_uint2(half2_of(left(f[0], x.x), left(f[1], x.y)), half2_of(left(f[2], y.x), left(f[3], y.y)));
            }
        }
        __syncthreads();
    }
};

// A lane's codes of a block of 16 keys: K rows lane / 4 and 8 more, 16 bytes of every 64; V rows 2 (lane % 4) and the next, and 8 more of both.
template <class F> struct KeyRegs { uint4 k[F::HDP / 64][2]; };
template <class F> struct ValueRegs { uint4 v[F::VG][4]; };

// A block on its way, 16 rows of keys and of values in the warp's part of a ring in shared memory.  The copies take whole rows, 512 bytes an
// instruction (with 64 bytes of every row, each lane copying what it reads, the copies alone took as long as everything together: 103 of
// 114 us, 64 sequences of up to 2,048 keys, 16 heads); a row's 16-byte chunks are stored at their number xor the row's, so that neither the
// reads of keys (8 lanes: two rows, four chunks of each) nor those of values (four rows, two chunks) meet in a bank.
template <int HDP> __device__ __forceinline__ int place_in(int row, int chunk) {
    return row * HDP + ((HDP == 64 ? chunk ^ ((row >> 1) & 3) : chunk ^ (row & 7)) * 16);
}
__device__ __forceinline__ void copy_async(uint32_t to, const uint8_t* from, bool there) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(to), "l"(from), "r"(there ? 16 : 0) : "memory");       // 0: zeros
}
template <class F>
__device__ __forceinline__ void copy_block(uint32_t at, const uint8_t* k, const uint8_t* v, int hd_) {
    constexpr int CPR = F::HDP / 16, ROWS = 32 / CPR;          // chunks a row, rows an instruction
    const int hd = F::EXACT ? F::HDP : hd_, lane = threadIdx.x & 31, row = lane / CPR, chunk = lane % CPR;
    const bool there = F::EXACT || chunk * 16 < hd;
    const uint32_t off = there ? row * hd + chunk * 16 : 0;
#pragma unroll
    for (int i = 0; i < C8_BLOCK / ROWS; ++i) {
        const uint32_t to = at + place_in<F::HDP>(row + i * ROWS, chunk), from = off + (there ? i * ROWS * hd : 0);
        copy_async(to, k + from, there);
        copy_async(to + C8_BLOCK * F::HDP, v + from, there);
    }
}
template <class F>
__device__ __forceinline__ void take_block(KeyRegs<F>& kr, ValueRegs<F>& vr, const uint8_t* at) {
    const int lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
#pragma unroll
    for (int j = 0; j < F::HDP / 64; ++j)
#pragma unroll
        for (int h = 0; h < 2; ++h) kr.k[j][h] = *reinterpret_cast<const uint4*>(at + place_in<F::HDP>(g + 8 * h, chunk_of<F::HDP>(j, t)));
    at += C8_BLOCK * F::HDP;
#pragma unroll
    for (int j = 0; j < F::VG; ++j)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            const int row = 2 * t + (r & 1) + 8 * (r >> 1);
            if (F::HDP == 64) {
                const uint2 x = *reinterpret_cast<const uint2*>(at + place_in<F::HDP>(row, g >> 1) + (g & 1) * 8);
                vr.v[j][r] = make_uint4(x.x, x.y, 0, 0);
            } else vr.v[j][r] = *reinterpret_cast<const uint4*>(at + place_in<F::HDP>(row, g + 8 * j));
        }
}
__device__ __forceinline__ uint32_t word(const uint4& v, int i) { return i == 0 ? v.x : i == 1 ? v.y : i == 2 ? v.z : v.w; }

// Sums of a block: s[nt] = {key g column 2t, key g column 2t + 1, key g + 8 ..}, without their factors.  One column tile: two chains of
// products, added at the end.  kept: the lane's part of the queries, where they stay in registers.
template <class F>
__device__ __forceinline__ void products(float (&s)[F::NT][4], const KeyRegs<F>& r, const Queries<F>& Q, const uint2* kept) {
    const int lane = threadIdx.x & 31;
    float odd[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int nt = 0; nt < F::NT; ++nt) s[nt][0] = s[nt][1] = s[nt][2] = s[nt][3] = 0.f;
#pragma unroll
    for (int j = 0; j < F::HDP / 64; ++j)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            uint32_t a0, a1, a2, a3;
            c8_half4(word(r.k[j][0], i), a0, a2);
            c8_half4(word(r.k[j][1], i), a1, a3);
#pragma unroll
            for (int nt = 0; nt < F::NT; ++nt)
#pragma unroll
                for (int p = 0; p < F::PARTS; ++p) {
                    const uint2 b = F::KEEP ? kept[j * 4 + i] : Q.b[p][nt][j * 4 + i][lane];
                    if (F::NT == 1 && ((i + p) & 1)) mma(odd, a0, a1, a2, a3, b.x, b.y);
                    else mma(s[nt], a0, a1, a2, a3, b.x, b.y);
                }
        }
    if (F::NT == 1) {
#pragma unroll
        for (int i = 0; i < 4; ++i) s[0][i] += odd[i];
    }
}

// Where a row of the step looks: the first of its places.
__device__ __forceinline__ int first_seen(int place, int window) { return window > 0 ? max(0, place + 1 - window) : 0; }

constexpr float LOWEST = -3.402823466e38f;       // a maximum over nothing
// Weights as float16 operands are times 2^WEIGHT_UP, and so are the sums of values until they are results.
constexpr float WEIGHT_UP = 14.f, WEIGHT_DOWN = 1.f / 16384.f;

// Scores of a step of single rows lie by key, a key's columns side by side in the next power of two (at most 16, or a multiple of 16).
__host__ __device__ __forceinline__ int score_columns(int per) { return per <= 2 ? per : per <= 4 ? 4 : per <= 8 ? 8 : (per + 15) / 16 * 16; }
// The sum over a key's columns of 2^(score - lse)
__device__ __forceinline__ float weight_of(const float* __restrict__ scores, const float* lse, int per) {
    float sum = 0.f;
    if (per <= 2) {
        sum = ex2(scores[0] - lse[0]);
        if (per == 2) sum += ex2(scores[1] - lse[1]);
        return sum;
    }
    for (int c = 0; c < per; c += 4) {
        const float4 v = *reinterpret_cast<const float4*>(scores + c);
        sum += ex2(v.x - lse[c]);
        if (c + 1 < per) sum += ex2(v.y - lse[c + 1]);
        if (c + 2 < per) sum += ex2(v.z - lse[c + 2]);
        if (c + 3 < per) sum += ex2(v.w - lse[c + 3]);
    }
    return sum;
}

// ---------------------------------------------------------------------------------------
// A range of the keys for a tile of columns.  partial: null, or [T * nh][ranges][hd + 4] for a second launch: the unnormalised sum (times
// 2^WEIGHT_UP), the maximum it is relative to, as what it lies above the denominator's, the denominator's maximum and the denominator.  scores: null, or (runs of one row) the base-2 scores of the
// tile's `per` columns, [n_seqs * nkv][score_stride][score_columns(per)].
// lse: null, or [T * nh], log2 of the denominator (where there is no second launch).  Several ranges without `partial`: they are the CTAs of a
// cluster, which join in their shared memory, each for its part of the result; with `weights` and scores each then adds up its own keys'
// weights (the tile has all the columns of its sequence and head then).
// ---------------------------------------------------------------------------------------
template <class F, bool CLUSTERED>
__device__ __forceinline__ void attend_tile(const Tile& T, int range, int ranges, const typename F::TA* __restrict__ q, const Cache8& c, const Step& S,
                                            typename F::TA* __restrict__ out, float* __restrict__ partial, float* __restrict__ scores, int score_stride,
                                            float* __restrict__ lse, float* __restrict__ weights) {
    constexpr int NT = F::NT, NC = F::NC, MT = F::MT, HDP = F::HDP;
    extern __shared__ __align__(16) uint8_t ring[];
    __shared__ Queries<F> Q;
    __shared__ float s_stat[WARPS][NC][3], s_ranks[CLUSTERED ? CLUSTER : 1][NC][3], s_lse[NC];
    float (*s_o)[NC][HDP + 4] = reinterpret_cast<float (*)[NC][HDP + 4]>(ring);        // [WARPS], once the keys are through
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3, hd = F::EXACT ? HDP : c.hd;
    // this range's blocks of 16 keys
    const int place0 = T.start + T.row(0), place1 = T.start + T.row(T.n - 1);
    const int block0 = first_seen(place0, S.window) / C8_BLOCK, blocks = place1 / C8_BLOCK + 1 - block0;
    const int each = (blocks + ranges * WARPS - 1) / (ranges * WARPS) * WARPS;
    const int from = block0 + range * each, to = min(from + each, block0 + blocks);

    // The blocks the warp still has to ask for: column of the page table and block of that page; the page is looked up one block ahead.
    const int per_page = c.page_size / C8_BLOCK;
    int ask = from + warp, column = ask / per_page, inner = ask - column * per_page, slot = 0;
    const int* pages = c.table + (size_t)T.seq * c.table_stride;
    auto page_at = [&](int col) { return TQ_CHECKED(pages[TQ_CHECKED(col, c.table_stride, TQ_IDX_TABLE_COLUMN)], c.n_pages, TQ_IDX_PAGE); };
    int page = ask < to ? page_at(column) : 0;
    uint32_t kbs[F::STAGES - 1], vbs[F::STAGES - 1];      // the bytes of the blocks on their way, oldest first
    const uint32_t mine = (uint32_t)__cvta_generic_to_shared(ring) + warp * (F::STAGES * F::STAGE_BYTES);
    // (a page's plane has fewer than 2^31 codes: c8_check)
    const uint32_t plane = (uint32_t)c.nkv * c.page_size * hd, plane_scales = (uint32_t)c.nkv * per_page;
    const uint8_t* codes_g = c.codes + (size_t)T.g * c.page_size * hd;
    const uint8_t* scales_g = c.scales + (size_t)T.g * per_page;
    auto next = [&](uint32_t& kb, uint32_t& vb) {
        if (ask < to) {
            const uint8_t* k = codes_g + (size_t)(uint32_t)page * (2u * plane) + (uint32_t)(inner * (C8_BLOCK * hd));
            copy_block<F>(mine + slot * F::STAGE_BYTES, k, k + plane, hd);
            const uint8_t* b8 = scales_g + (size_t)(uint32_t)page * (2u * plane_scales) + inner;
            kb = *b8;
            vb = b8[plane_scales];
            ask += WARPS;
            inner += WARPS;
            const int was = column;
            while (inner >= per_page) { inner -= per_page; ++column; }
            if (column != was && ask < to) page = page_at(column);
        }
        asm volatile("cp.async.commit_group;" ::: "memory");
        slot = slot + 1 == F::STAGES ? 0 : slot + 1;
    };
#pragma unroll
    for (int i = 0; i < F::STAGES - 1; ++i) { kbs[i] = vbs[i] = 1; next(kbs[i], vbs[i]); }

    Q.load(q, T, S, hd);
    int place_of[NT][2];               // the lane's columns' places
    float f[NT][2];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            place_of[nt][j] = Q.place[nt * 8 + 2 * t + j];
            f[nt][j] = Q.factor[nt * 8 + 2 * t + j];
        }
    uint2 kept[F::KEEP ? F::STEPS : 1];
    if (F::KEEP) {
#pragma unroll
        for (int i = 0; i < F::STEPS; ++i) kept[F::KEEP ? i : 0] = Q.b[0][0][i][lane];
    }
    float o[NT][MT][4], m[NT][2], mo[NT][2], l[NT][2];        // m: maximum of the scores, mo: that of scores and value scales, less m
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
        for (int i = 0; i < MT; ++i) o[nt][i][0] = o[nt][i][1] = o[nt][i][2] = o[nt][i][3] = 0.f;
        m[nt][0] = m[nt][1] = mo[nt][0] = mo[nt][1] = LOWEST;
        l[nt][0] = l[nt][1] = 0.f;
    }
    const int score_cols = score_columns(T.per);
    float* own_scores = scores != nullptr ? scores + ((size_t)T.seq * c.nkv + T.g) * score_stride * score_cols : nullptr;
    int taken = 0;
#pragma unroll 1
    for (int b = from + warp; b < to; b += WARPS) {
        asm volatile("cp.async.wait_group %0;" ::"n"(F::STAGES - 2) : "memory");
        KeyRegs<F> kc;
        ValueRegs<F> vc;
        __syncwarp();                  // each lane's copies of this block are there, so all of them
        take_block<F>(kc, vc, ring + warp * (F::STAGES * F::STAGE_BYTES) + taken * F::STAGE_BYTES);
        taken = taken + 1 == F::STAGES ? 0 : taken + 1;
        __syncwarp();                  // all lanes have read the block before this one, whose place is filled next
        const float ks = c8_scale(kbs[0]), ve = (float)((int)vbs[0] - 127);
#pragma unroll
        for (int i = 0; i + 1 < F::STAGES - 1; ++i) { kbs[i] = kbs[i + 1]; vbs[i] = vbs[i + 1]; }
        next(kbs[F::STAGES - 2], vbs[F::STAGES - 2]);
        float s[NT][4];
        products<F>(s, kc, Q, kept);
        const int key = b * C8_BLOCK + g;
        // every column sees all 16 keys? (those that are not there may see them too: nobody reads their sums)
        const bool whole = b * C8_BLOCK + C8_BLOCK - 1 <= place0 && (S.window <= 0 || b * C8_BLOCK > place1 - S.window);
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
            const float f0 = f[nt][0] * ks, f1 = f[nt][1] * ks;
            s[nt][0] *= f0; s[nt][1] *= f1; s[nt][2] *= f0; s[nt][3] *= f1;
        }
        if (!whole) {
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const int p = place_of[nt][j & 1], k = key + 8 * (j >> 1);
                    if (k > p || (S.window > 0 && k <= p - S.window)) s[nt][j] = -INFINITY;
                }
        }
        if (scores != nullptr) {
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    const int col = T.first + nt * 8 + 2 * t, k = key + 8 * h;
                    if (nt * 8 + 2 * t >= T.n || k >= score_stride) continue;
                    float* to = own_scores + (size_t)k * score_cols + col;
                    if (score_cols > 1) *reinterpret_cast<float2*>(to) = make_float2(s[nt][2 * h], s[nt][2 * h + 1]);
                    else *to = s[nt][2 * h];
                }
        }
        // the maxima grow now and then: found by all lanes of a column together when one of them sees a larger value
        float top[NT][2];
        bool grows = false;
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                top[nt][j] = fmaxf(s[nt][j], s[nt][j + 2]);
                grows |= top[nt][j] > m[nt][j] || top[nt][j] - m[nt][j] + ve > mo[nt][j];
            }
        if (__any_sync(0xffffffffu, grows)) {
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                for (int j = 0; j < 2; ++j) {
#pragma unroll
                    for (int x = 4; x < 32; x <<= 1) top[nt][j] = fmaxf(top[nt][j], __shfl_xor_sync(0xffffffffu, top[nt][j], x));
                    const float mn = fmaxf(m[nt][j], top[nt][j]), up = m[nt][j] - mn, was = mo[nt][j] + up, mon = fmaxf(was, top[nt][j] - mn + ve);
                    l[nt][j] *= ex2(up);
                    m[nt][j] = mn;
                    if (mon > was) {
                        const float down = ex2(was - mon);
#pragma unroll
                        for (int i = 0; i < MT; ++i) { o[nt][i][j] *= down; o[nt][i][j + 2] *= down; }
                    }
                    mo[nt][j] = mon;
                }
        }
        uint32_t p_hi[NT][2], p_lo[NT][2];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
            float w[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const float below = s[nt][j] - m[nt][j & 1];
                l[nt][j & 1] += ex2(below);
                w[j] = ex2(below + (ve + WEIGHT_UP - mo[nt][j & 1]));
            }
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const uint32_t hi = half2_of(w[2 * h], w[2 * h + 1]);
                p_hi[nt][h] = transpose8x8(hi);
                if (F::PARTS == 2) {
                    const float2 x = float2_of(hi);
                    p_lo[nt][h] = transpose8x8(half2_of(w[2 * h] - x.x, w[2 * h + 1] - x.y));
                }
            }
        }
        // Values no column may see come with a weight of 0, which does not remove a NaN: such codes are taken out of the product, and put
        // back as NaN into the sums of the columns that do see the key.
        uint32_t lost[F::VG][4] = {};                          // of the lane's four rows: which of its 16 elements are NaN
        bool some = false;
        if (!whole) {
#pragma unroll
            for (int j = 0; j < F::VG; ++j)
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    uint32_t u[4] = {vc.v[j][k].x, vc.v[j][k].y, vc.v[j][k].z, vc.v[j][k].w};
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const uint32_t hit = ((u[i] & 0x7f7f7f7fu) + 0x01010101u) & 0x80808080u;     // the top bit of every byte 0x7f or 0xff
                        lost[j][k] |= ((hit >> 7 & 1u) | (hit >> 14 & 2u) | (hit >> 21 & 4u) | (hit >> 28 & 8u)) << (4 * i);
                        u[i] &= ~((hit >> 7) * 0xffu);
                    }
                    vc.v[j][k] = make_uint4(u[0], u[1], u[2], u[3]);
                    some |= lost[j][k] != 0;
                }
            some = __any_sync(0xffffffffu, some);
        }
#pragma unroll
        for (int i = 0; i < MT; i += 2) {
            // words i / 2 of the lane's four rows: two steps of 16 elements
            const int j = HDP > 128 ? i / 8 : 0, wd = (i - 8 * j) / 2;
            const uint32_t r0 = word(vc.v[j][0], wd), r1 = word(vc.v[j][1], wd), r2 = word(vc.v[j][2], wd), r3 = word(vc.v[j][3], wd);
            uint32_t a0, a1, a2, a3, e0, e1, e2, e3;
            c8_half4(__byte_perm(r0, r1, 0x5140), a0, a1);
            c8_half4(__byte_perm(r2, r3, 0x5140), a2, a3);
            c8_half4(__byte_perm(r0, r1, 0x7362), e0, e1);
            c8_half4(__byte_perm(r2, r3, 0x7362), e2, e3);
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
                mma(o[nt][i], a0, a1, a2, a3, p_hi[nt][0], p_hi[nt][1]);
                mma(o[nt][i + 1], e0, e1, e2, e3, p_hi[nt][0], p_hi[nt][1]);
                if (F::PARTS == 2) {
                    mma(o[nt][i], a0, a1, a2, a3, p_lo[nt][0], p_lo[nt][1]);
                    mma(o[nt][i + 1], e0, e1, e2, e3, p_lo[nt][0], p_lo[nt][1]);
                }
            }
        }
        if (some) {
#pragma unroll 1
            for (int k16 = 0; k16 < C8_BLOCK; ++k16) {
                const int owner = (lane & ~3) | ((k16 & 7) >> 1), slot16 = (k16 & 1) + 2 * (k16 >> 3);
#pragma unroll
                for (int j = 0; j < F::VG; ++j) {
                    const uint32_t own = slot16 == 0 ? lost[j][0] : slot16 == 1 ? lost[j][1] : slot16 == 2 ? lost[j][2] : lost[j][3];
                    const uint32_t bits = __shfl_sync(0xffffffffu, own, owner);
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
    asm volatile("cp.async.wait_group 0;" ::: "memory");
    __syncthreads();                   // every warp is through with its part of the ring
    // the warps' sums together
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            const int col = nt * 8 + 2 * t + j;
#pragma unroll
            for (int x = 4; x < 32; x <<= 1) l[nt][j] += __shfl_xor_sync(0xffffffffu, l[nt][j], x);
            if (col >= T.n) continue;
            if (g == 0) { s_stat[warp][col][0] = mo[nt][j]; s_stat[warp][col][1] = m[nt][j]; s_stat[warp][col][2] = l[nt][j]; }
#pragma unroll
            for (int i = 0; i < MT; ++i) {
                const int d = HDP == 64 ? g * 8 + 2 * i : (i / 8) * 128 + g * 16 + 2 * (i % 8);
                *reinterpret_cast<float2*>(&s_o[warp][col][d]) = make_float2(o[nt][i][j], o[nt][i][j + 2]);
            }
        }
    __syncthreads();
    for (int col = warp; col < T.n; col += WARPS) {
        float mw[WARPS], M = LOWEST, MO = LOWEST, L = 0.f;            // (MO: less M)
#pragma unroll
        for (int w = 0; w < WARPS; ++w) M = fmaxf(M, s_stat[w][col][1]);
#pragma unroll
        for (int w = 0; w < WARPS; ++w) MO = fmaxf(MO, s_stat[w][col][1] - M + s_stat[w][col][0]);
#pragma unroll
        for (int w = 0; w < WARPS; ++w) {
            const float below = s_stat[w][col][1] - M;
            mw[w] = exp2f(below + s_stat[w][col][0] - MO);
            L += s_stat[w][col][2] * exp2f(below);
        }
        if (CLUSTERED) {
            for (int d = lane; d < hd; d += 32) {
                float sum = 0.f;
#pragma unroll
                for (int w = 0; w < WARPS; ++w) sum += s_o[w][col][d] * mw[w];
                s_o[0][col][d] = sum;
            }
            __syncwarp();
            if (lane == 0) { s_stat[0][col][0] = MO; s_stat[0][col][1] = M; s_stat[0][col][2] = L; }
            continue;
        }
        const size_t at = Q.row[col];
        float* pp = partial != nullptr ? partial + (at * ranges + range) * (hd + 4) : nullptr;
        const float norm = exp2f(MO) / L;
        for (int d = lane; d < hd; d += 32) {
            float sum = 0.f;
#pragma unroll
            for (int w = 0; w < WARPS; ++w) sum += s_o[w][col][d] * mw[w];
            if (pp != nullptr) pp[d] = sum;
            else out[at * hd + d] = tq_from_float<typename F::TA>(sum * WEIGHT_DOWN * norm);
        }
        if (pp != nullptr && lane == 0) { pp[hd] = MO; pp[hd + 1] = M; pp[hd + 2] = L; }
        if (pp == nullptr && lse != nullptr && lane == 0) lse[at] = M + log2f(L);
    }
    if (!CLUSTERED) return;
    __syncwarp();
    // the cluster's sums together: statistics of all ranges first, then every CTA its part of the tile's results
    asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
    auto remote = [](const float* own, int rank) {
        uint32_t a;
        float v;
        asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(a) : "r"((uint32_t)__cvta_generic_to_shared(own)), "r"(rank));
        asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(a) : "memory");
        return v;
    };
    // (a thread's first element of every range is asked for beside the statistics, whose way is as long: one chat of 700 rows in 6 ranges 6.2 us, one
    // behind the other 6.8)
    const int element0 = range * WARPS * 32 + (int)threadIdx.x;
    float v[CLUSTER];
    auto fetch = [&](int i) {
#pragma unroll
        for (int r = 0; r < CLUSTER; ++r) v[r] = r < ranges ? remote(&s_o[0][i / hd][i % hd], r) : 0.f;
    };
    if (element0 < T.n * hd) fetch(element0);
    for (int i = threadIdx.x; i < ranges * NC * 3; i += WARPS * 32)
        if (i / 3 % NC < T.n) (&s_ranks[0][0][0])[i] = remote(&s_stat[0][0][0] + i % (NC * 3), i / (NC * 3));
    __syncthreads();
    // a column's denominator and, for each range, the factor of its sums
    auto join = [&](int col, float (&factors)[CLUSTER], float& MO, float& log_sum) {
        float M = LOWEST, L = 0.f;
        MO = LOWEST;
#pragma unroll
        for (int r = 0; r < CLUSTER; ++r) if (r < ranges) M = fmaxf(M, s_ranks[r][col][1]);
#pragma unroll
        for (int r = 0; r < CLUSTER; ++r) {
            factors[r] = LOWEST;
            if (r >= ranges) continue;
            const float below = s_ranks[r][col][1] - M;
            factors[r] = below + s_ranks[r][col][0];
            MO = fmaxf(MO, factors[r]);
            L += s_ranks[r][col][2] * ex2(below);
        }
#pragma unroll
        for (int r = 0; r < CLUSTER; ++r) factors[r] = ex2(factors[r] - MO);
        log_sum = M + log2f(L);
        return L;
    };
    float factors[CLUSTER], MO, log_sum;
    for (int i = element0; i < T.n * hd; i += ranges * WARPS * 32) {
        const int col = i / hd, d = i - col * hd;
        if (i != element0) fetch(i);
        const float L = join(col, factors, MO, log_sum);
        float sum = 0.f;
#pragma unroll
        for (int r = 0; r < CLUSTER; ++r) sum += v[r] * factors[r];
        out[Q.row[col] * hd + d] = tq_from_float<typename F::TA>(sum * WEIGHT_DOWN * (exp2f(MO) / L));
        if (lse != nullptr && d == 0) lse[Q.row[col]] = log_sum;
    }
    if (weights != nullptr) {
        if (threadIdx.x < T.n) {
            join(threadIdx.x, factors, MO, log_sum);
            s_lse[threadIdx.x] = log_sum;
        }
        __syncthreads();
        // (the step has one row of the sequence: it sees up to its own place)
        const int last = min(min(to * C8_BLOCK, place1 + 1), score_stride);
#pragma unroll 2
        for (int k = from * C8_BLOCK + threadIdx.x; k < last; k += WARPS * 32) {
            if (S.window > 0 && k + S.window <= T.start) continue;
            float* w = weights + ((size_t)c.page_of(T.seq, k) * c.nkv + T.g) * c.page_size + c.row(k);
            const float was = k < T.start ? *w : 0.f;
            *w = was + weight_of(own_scores + (size_t)k * score_cols, s_lse, T.per);
        }
    }
    // nobody leaves while its sums are being read
    asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}

template <class F, bool CLUSTERED>
__global__ void __launch_bounds__(WARPS * 32, F::PER_SM) attention8_kernel(const typename F::TA* __restrict__ q, Cache8 c, Step S, typename F::TA* __restrict__ out,
                                                                                           float* __restrict__ partial, float* __restrict__ scores, int score_stride,
                                                                                           float* __restrict__ lse, float* __restrict__ weights, int ranges) {
    tq_grid_wait();                    // everything below may read what the previous kernel wrote
    q = tq_fresh(q);
    tq_grid_launch_dependents();
    const int tile = blockIdx.x / ranges, tile_no = tile / c.nkv;
    const Tile T = tile_of(S, blockIdx.z, tile - tile_no * c.nkv, c.nkv, tile_no, F::NC);
    if (T.n > 0) attend_tile<F, CLUSTERED>(T, blockIdx.x - tile * ranges, ranges, q, c, S, out, partial, scores, score_stride, lse, weights);
}

// The prompt kernel gives values that a row may not see a weight of 0, which does not remove a NaN: key/value heads of sequences in whose pages
// `lost` [n_seqs][nkv][pages] marks such values are done again here, all others cost a look at their marks.
template <class F>
__global__ void __launch_bounds__(WARPS * 32) repair8_kernel(const typename F::TA* __restrict__ q, Cache8 c, Step S, typename F::TA* __restrict__ out,
                                                             const uint8_t* __restrict__ lost, int lost_stride, int page_size) {
    tq_grid_wait();                    // everything below may read what the previous kernel wrote
    q = tq_fresh(q);
    tq_grid_launch_dependents();
    const int seq = blockIdx.z, g = blockIdx.y, start = S.held[seq], run = S.cu_seqlens[seq + 1] - S.cu_seqlens[seq];
    if (run <= 0) return;
    const uint8_t* marks = lost + ((size_t)seq * c.nkv + g) * lost_stride;
    bool some = false;
    for (int p = first_seen(start, S.window) / page_size + (int)threadIdx.x; p <= (start + run - 1) / page_size; p += WARPS * 32) some |= marks[p] != 0;
    if (!__syncthreads_or(some)) return;
    for (int tile_no = blockIdx.x; ; tile_no += gridDim.x) {
        const Tile T = tile_of(S, seq, g, c.nkv, tile_no, F::NC);
        if (T.n <= 0) return;
        __syncthreads();
        attend_tile<F, false>(T, 0, 1, q, c, S, out, nullptr, nullptr, 0, nullptr, nullptr);
    }
}

// ---------------------------------------------------------------------------------------
// The ranges of a row joined, a block per row.  Blocks behind the rows' add the weights up from the scores the first launch left, 128 places
// of a (sequence, key/value head) each.
// ---------------------------------------------------------------------------------------
constexpr int JOIN_RANGES = 64;

// The statistics of row `at` of q (MO: less M), and each range's factor in s_f[0 .. ranges - 1]; by a warp, which then has them.
__device__ __forceinline__ void join_stats(const float* __restrict__ partial, size_t at, int ranges, int hd, float& MO, float& M, float& L, float* s_f) {
    const int lane = threadIdx.x & 31;
    const float* p = partial + at * ranges * (hd + 4) + hd;
    float mo[JOIN_RANGES / 32], m[JOIN_RANGES / 32], l[JOIN_RANGES / 32];
    MO = LOWEST; M = LOWEST; L = 0.f;
#pragma unroll
    for (int i = 0; i < JOIN_RANGES / 32; ++i) {
        const int r = lane + 32 * i;
        mo[i] = m[i] = LOWEST;
        l[i] = 0.f;
        if (r < ranges) { mo[i] = p[(size_t)r * (hd + 4)]; m[i] = p[(size_t)r * (hd + 4) + 1]; l[i] = p[(size_t)r * (hd + 4) + 2]; }
        M = fmaxf(M, m[i]);
    }
    M = tq_warp_max(M);
#pragma unroll
    for (int i = 0; i < JOIN_RANGES / 32; ++i) MO = fmaxf(MO, m[i] - M + mo[i]);
    MO = tq_warp_max(MO);
#pragma unroll
    for (int i = 0; i < JOIN_RANGES / 32; ++i) {
        L += l[i] * exp2f(m[i] - M);
        if (s_f != nullptr && lane + 32 * i < ranges) s_f[lane + 32 * i] = exp2f(m[i] - M + mo[i] - MO);
    }
    L = tq_warp_sum(L);
}

template <typename TA>
__global__ void __launch_bounds__(128) join8_kernel(Cache8 c, Step S, const float* __restrict__ partial, int ranges, TA* __restrict__ out, int rows,
                                                    float* __restrict__ lse, const float* __restrict__ scores, int score_stride, float* __restrict__ weights) {
    tq_grid_wait();                    // everything below may read what the previous kernel wrote
    tq_grid_launch_dependents();
    __shared__ float s_f[JOIN_RANGES], s_lse[128 + 4];
    const int seq = blockIdx.z, g = blockIdx.y, per = S.nh / c.nkv, hd = c.hd, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int t_begin = S.cu_seqlens[seq], run = S.cu_seqlens[seq + 1] - t_begin, columns = run * per;
    auto query = [&](int col) { const int r = col / per; return (size_t)(t_begin + r) * S.nh + g * per + (col - r * per); };
    if ((int)blockIdx.x < rows) {
        if ((int)blockIdx.x >= columns) return;
        const size_t at = query(blockIdx.x);
        const float* p = partial + at * ranges * (hd + 4);
        float v[2][8];                 // the first ranges' elements, asked for beside the statistics
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
            for (int r = 0; r < 8; ++r) v[h][r] = r < ranges && (int)threadIdx.x + 128 * h < hd ? p[(size_t)r * (hd + 4) + threadIdx.x + 128 * h] : 0.f;
        if (warp == 0) {
            float MO, M, L;
            join_stats(partial, at, ranges, hd, MO, M, L, s_f);
            if (lane == 0) {
                s_lse[0] = exp2f(MO) / L;
                if (lse != nullptr) lse[at] = M + log2f(L);
            }
        }
        __syncthreads();
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const int d = threadIdx.x + 128 * h;
            if (d >= hd) break;
            float sum = 0.f;
#pragma unroll
            for (int r = 0; r < 8; ++r) if (r < ranges) sum += v[h][r] * s_f[r];
#pragma unroll 8
            for (int r = 8; r < ranges; ++r) sum += p[(size_t)r * (hd + 4) + d] * s_f[r];
            out[at * hd + d] = tq_from_float<TA>(sum * WEIGHT_DOWN * s_lse[0]);
        }
        return;
    }
    // (the step has one row of the sequence: it sees up to its own place)
    const int start = S.held[seq], place0 = ((int)blockIdx.x - rows) * 128, place = place0 + (int)threadIdx.x;
    if (run <= 0 || place0 > start) return;
    float sum = 0.f;
    for (int c0 = 0; c0 < per; c0 += 128) {
        const int n = min(128, per - c0);
        __syncthreads();
        for (int x = warp; x < n; x += 4) {
            float MO, M, L;
            join_stats(partial, query(c0 + x), ranges, hd, MO, M, L, nullptr);
            if (lane == 0) s_lse[x] = M + log2f(L);
        }
        __syncthreads();
        if (place <= start && place < score_stride)
            sum += weight_of(scores + (((size_t)seq * c.nkv + g) * score_stride + place) * score_columns(per) + c0, s_lse, n);
    }
    if (place > start || place >= score_stride || (S.window > 0 && place + S.window <= start)) return;
    float* w = weights + ((size_t)c.page_of(seq, place) * c.nkv + g) * c.page_size + c.row(place);
    *w = (place < start ? *w : 0.f) + sum;
}

// ---------------------------------------------------------------------------------------
// Sums of weights from the queries and the keys again.  A CTA has KB blocks of 16 keys of a (sequence, key/value head); each of its four warps
// holds all of them as left operands and walks every fourth tile of 8 columns that see them, whose queries go from memory straight to its
// registers: no shared memory, no barrier but the one at the end, where the warps' sums meet in order.  One writer per sum: the same bits
// every time.  (A warp per block and the columns one tile after another through shared memory: 588 rows of 8 heads of 256 484 us.)
// ---------------------------------------------------------------------------------------
// sixteen elements of a row; the row's offset is a multiple of 16 elements
__device__ __forceinline__ void load16(float (&x)[16], const __nv_bfloat16* p, bool aligned) {
    if (aligned) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const uint4 v = reinterpret_cast<const uint4*>(p)[h];
            const uint32_t u[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
            for (int e = 0; e < 4; ++e) { x[8 * h + 2 * e] = __uint_as_float(u[e] << 16); x[8 * h + 2 * e + 1] = __uint_as_float(u[e] & 0xffff0000u); }
        }
    } else {
#pragma unroll
        for (int e = 0; e < 16; ++e) x[e] = tq_to_float(p[e]);
    }
}
__device__ __forceinline__ void load16(float (&x)[16], const float* p, bool aligned) {
    if (aligned) {
#pragma unroll
        for (int h = 0; h < 4; ++h) {
            const float4 v = reinterpret_cast<const float4*>(p)[h];
            x[4 * h] = v.x; x[4 * h + 1] = v.y; x[4 * h + 2] = v.z; x[4 * h + 3] = v.w;
        }
    } else {
#pragma unroll
        for (int e = 0; e < 16; ++e) x[e] = p[e];
    }
}

template <class F, int KB>
__global__ void __launch_bounds__(WARPS * 32) weigh8_kernel(const typename F::TA* __restrict__ q, Cache8 c, Step S, const float* __restrict__ lse, float* __restrict__ weights) {
    tq_grid_wait();                    // everything below may read what the previous kernel wrote
    q = tq_fresh(q);
    tq_grid_launch_dependents();
    using TA = typename F::TA;
    constexpr int KEYS = KB * C8_BLOCK;
    const bool aligned = ((uintptr_t)q & 15) == 0;
    __shared__ float s_sum[WARPS][KEYS];
    const int seq = blockIdx.z, gh = blockIdx.y, warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3, hd = c.hd;
    const Tile T = tile_of(S, seq, gh, c.nkv, 0, 8);
    const int key0 = blockIdx.x * KEYS, end = T.start + T.run;
    // rows of the run that see some of the CTA's keys
    const int row0 = max(0, key0 - T.start), row1 = S.window > 0 ? min(T.run, key0 + KEYS - 1 + S.window - T.start) : T.run;
    if (row0 >= row1) return;
    uint4 kr[KB][F::HDP / 64][2];
    float ks[KB];
#pragma unroll
    for (int b = 0; b < KB; ++b) {
        const int key = key0 + b * C8_BLOCK;
        ks[b] = 0.f;
        // blocks behind the last row, or whose pages may have been given back, have no page
        const bool there = key < end && !(S.window > 0 && key + C8_BLOCK - 1 + S.window <= T.start);
        const int page = there ? c.page_of(seq, key) : 0, row = c.row(key);
        const uint8_t* k = c.codes + c.codes_at(page, 0, gh) + (size_t)row * hd;
#pragma unroll
        for (int j = 0; j < F::HDP / 64; ++j)
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const int at = chunk_of<F::HDP>(j, t) * 16;
                kr[b][j][h] = there && at < hd ? *reinterpret_cast<const uint4*>(k + (g + 8 * h) * hd + at) : make_uint4(0, 0, 0, 0);
            }
        if (there) ks[b] = c8_scale(c.scales[c.scales_at(page, 0, gh) + row / C8_BLOCK]);
    }
    float sum[KB][2] = {};
    const int last = row1 * T.per;
    for (int first = row0 * T.per + warp * 8; first < last; first += WARPS * 8) {
        // the lane's column: its queries, scaled to a largest element between 2^14 and 2^15, and what its scores need
        const int col = first + g;
        const bool mine = col < last;
        const size_t at = mine ? T.query(col, S) : 0;
        float x[F::HDP / 64][16];
        uint32_t top = 0;
#pragma unroll
        for (int j = 0; j < F::HDP / 64; ++j) {
            const int d = chunk_of<F::HDP>(j, t) * 16;
#pragma unroll
            for (int e = 0; e < 16; ++e) x[j][e] = 0.f;
            if (mine && d < hd) load16(x[j], q + at * hd + d, aligned);
#pragma unroll
            for (int e = 0; e < 16; ++e) top = max(top, c8_magnitude(x[j][e]));
        }
        top = max(top, __shfl_xor_sync(0xffffffffu, top, 1));
        top = max(top, __shfl_xor_sync(0xffffffffu, top, 2));
        const int shift = min(126, 14 - max((int)(top >> 23) - 127, -126));
        const float up = __uint_as_float((uint32_t)(127 + shift) << 23), factor = S.factor * __uint_as_float((uint32_t)(127 - shift) << 23);
        const float minus = mine ? -lse[at] : 0.f;
        const int place = mine ? T.start + T.row(col) : -1;               // (T.first is 0)
        uint2 b0[F::HDP / 64][4], b1[F::PARTS == 2 ? F::HDP / 64 : 1][4];
#pragma unroll
        for (int j = 0; j < F::HDP / 64; ++j)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                float v[4];
#pragma unroll
                for (int e = 0; e < 4; ++e) v[e] = x[j][4 * i + e] * up;
                b0[j][i] = make_uint2(half2_of(v[0], v[1]), half2_of(v[2], v[3]));
                if (F::PARTS == 2) {
                    const float2 p = float2_of(b0[j][i].x), r = float2_of(b0[j][i].y);
                    auto left = [](float a, float h) { const float d = a - h; return fabsf(d) < INFINITY ? d : 0.f; };
                    b1[F::PARTS == 2 ? j : 0][i] = make_uint2(half2_of(left(v[0], p.x), left(v[1], p.y)), half2_of(left(v[2], r.x), left(v[3], r.y)));
                }
            }
        // what the lane's two columns of results need, from the lanes that have them
        float f[2], m[2];
        int p[2];
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            const int from = (2 * t + j) * 4;
            f[j] = __shfl_sync(0xffffffffu, factor, from);
            m[j] = __shfl_sync(0xffffffffu, minus, from);
            p[j] = __shfl_sync(0xffffffffu, place, from);
        }
#pragma unroll
        for (int b = 0; b < KB; ++b) {
            float s[4] = {}, odd[4] = {};
#pragma unroll
            for (int j = 0; j < F::HDP / 64; ++j)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    uint32_t a0, a1, a2, a3;
                    c8_half4(word(kr[b][j][0], i), a0, a2);
                    c8_half4(word(kr[b][j][1], i), a1, a3);
                    mma(i & 1 ? odd : s, a0, a1, a2, a3, b0[j][i].x, b0[j][i].y);
                    if (F::PARTS == 2) mma(i & 1 ? s : odd, a0, a1, a2, a3, b1[F::PARTS == 2 ? j : 0][i].x, b1[F::PARTS == 2 ? j : 0][i].y);
                }
#pragma unroll
            for (int j = 0; j < 2; ++j)
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    const int k = key0 + b * C8_BLOCK + g + 8 * h;
                    if (k <= p[j] && (S.window <= 0 || k > p[j] - S.window)) sum[b][h] += ex2(fmaf(s[j + 2 * h] + odd[j + 2 * h], f[j] * ks[b], m[j]));
                }
        }
    }
#pragma unroll
    for (int b = 0; b < KB; ++b)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            sum[b][h] += __shfl_xor_sync(0xffffffffu, sum[b][h], 1);
            sum[b][h] += __shfl_xor_sync(0xffffffffu, sum[b][h], 2);
            if (t == 0) s_sum[warp][b * C8_BLOCK + g + 8 * h] = sum[b][h];
        }
    __syncthreads();
    const int k = key0 + (int)threadIdx.x;
    if (threadIdx.x < KEYS && k < end && !(S.window > 0 && k + S.window <= T.start)) {       // (others: no row of the step sees them)
        float all = 0.f;
#pragma unroll
        for (int w = 0; w < WARPS; ++w) all += s_sum[w][threadIdx.x];
        float* w = weights + ((size_t)c.page_of(seq, k) * c.nkv + gh) * c.page_size + c.row(k);
        *w = (k < T.start ? *w : 0.f) + all;
    }
}

template <class F>
int launch_repair8(const void* q, const Cache8& c, const Step& S, void* out, const void* lost, int lost_stride, int n_seqs, cudaStream_t stream) {
    static std::atomic<unsigned long long> asked{0};
    const cudaError_t e = tq_reserve_smem(repair8_kernel<F>, F::SMEM, asked);
    if (e != cudaSuccess) TQ_FAIL(-1, "repair8: cannot reserve %d bytes of shared memory: %s", F::SMEM, cudaGetErrorString(e));
    const int heads = c.nkv * n_seqs, each = heads >= 444 ? 1 : 444 / heads;
    tq_launch(dim3(each, c.nkv, n_seqs), WARPS * 32, F::SMEM, stream)(repair8_kernel<F>, (const typename F::TA*)q, c, S, (typename F::TA*)out, (const uint8_t*)lost, lost_stride, c.page_size);
    TQ_CHECK_LAUNCH("repair8");
    return 0;
}
template <class F>
int launch8(const void* q, const Cache8& c, const Step& S, void* out, float* partial, int ranges, float* scores, int score_stride, float* lse, float* weights,
            int n_seqs, int max_q_len, cudaStream_t stream) {
    const long long tiles = ((long long)max_q_len * (S.nh / c.nkv) + F::NC - 1) / F::NC * c.nkv;
    TQ_REQUIRE(tiles * ranges < (1ll << 31), "attention8: runs of %d rows", max_q_len);
    TQ_REQUIRE(weights == nullptr || tiles == c.nkv, "attention8: a tile of %d columns does not hold %d query heads", F::NC, S.nh / c.nkv);
    auto launch = [&](auto kernel, std::atomic<unsigned long long>& asked, int cluster) -> int {
        const cudaError_t e = tq_reserve_smem(kernel, F::SMEM, asked);
        if (e != cudaSuccess) TQ_FAIL(-1, "attention8: cannot reserve %d bytes of shared memory: %s", F::SMEM, cudaGetErrorString(e));
        tq_launch(dim3((unsigned)(tiles * ranges), 1, n_seqs), WARPS * 32, F::SMEM, stream, cluster)(
            kernel, (const typename F::TA*)q, c, S, (typename F::TA*)out, partial, scores, score_stride, lse, weights, ranges);
        return 0;
    };
    static std::atomic<unsigned long long> asked{0}, asked_clustered{0};
    const int rc = ranges > 1 && partial == nullptr ? launch(attention8_kernel<F, true>, asked_clustered, ranges) : launch(attention8_kernel<F, false>, asked, 1);
    if (rc) return rc;
    TQ_CHECK_LAUNCH("attention8");
    return 0;
}
template <class F, int KB>
int launch_weigh8(const void* q, const Cache8& c, const Step& S, const float* lse, float* weights, int n_seqs, int max_kv_len, cudaStream_t stream) {
    const int per_cta = KB * C8_BLOCK;
    tq_launch(dim3((max_kv_len + per_cta - 1) / per_cta, c.nkv, n_seqs), WARPS * 32, 0, stream)(weigh8_kernel<F, KB>, (const typename F::TA*)q, c, S, lse, weights);
    TQ_CHECK_LAUNCH("weigh8");
    return 0;
}
// Two tiles of 8 columns where there are more than 8 (heads of up to 128: beyond, the sums of 16 columns do not fit the registers)
#define C8_FORMS(columns, CALL)                                                                                              \
    do {                                                                                                                     \
        if (hd == 128) { if ((columns) > 8) return CALL(128, 2, true); return CALL(128, 1, true); }                          \
        if (hd == 64) { if ((columns) > 8) return CALL(64, 2, true); return CALL(64, 1, true); }                             \
        if (hd < 64) { if ((columns) > 8) return CALL(64, 2, false); return CALL(64, 1, false); }                            \
        if (hd < 128) { if ((columns) > 8) return CALL(128, 2, false); return CALL(128, 1, false); }                         \
        return CALL(256, 1, false);                                                                                          \
    } while (0)

int check_step(const char* what, int nh, int nkv, int n_seqs, int longest, int window) {
    TQ_REQUIRE(nh >= 1 && nh % nkv == 0 && nkv <= 65535, "%s: %d heads are not a multiple of %d key/value heads", what, nh, nkv);
    TQ_REQUIRE(n_seqs <= 65535 && longest >= 1 && window >= 0, "%s: %d sequences, longest %d, window %d", what, n_seqs, longest, window);
    return 0;
}

}  // namespace

// q [T, nh, hd], out [T, nh * hd]; place i sees j <= i with window == 0 or i - j < window.  max_q_len: the longest run.  ranges > 1: the keys
// of a row are cut into that many ranges, which join as a cluster (up to 8; partial null) or in a second launch (up to 64; partial
// [T * nh * ranges * (hd + 4)]).  lse [T, nh] float32 or null.  scores [n_seqs * nkv, score_stride, score_columns(nh / nkv)] with weights [n_pages,
// nkv, page_size], or both null: the weights of a step of single rows are added up by whoever joins, so by clusters only of all of a key/value
// head's query heads, and of two ranges or more.  score_stride: at least max_kv_len, the longest held[s] + run.
struct Attention8Call {
    const void *q, *codes, *scales;
    const int *cu_seqlens, *held, *page_table;
    void* out;
    float *partial, *lse, *scores, *weights;
    cudaStream_t stream;
    int act_dtype, table_stride, page_size, window, ranges, score_stride, max_kv_len, n_pages, n_seqs, max_q_len, nh, nkv, hd;
    float scale;
};
TQ_EXPORT int tq_attention8(const void* packed, int bytes) {
    C8_REQUIRE_CALL("attention8", Attention8Call);
    const Attention8Call x = c8_call<Attention8Call>(packed);
    const void* q = x.q;
    float *partial = x.partial, *scores = x.scores, *weights = x.weights;
    const int page_size = x.page_size, window = x.window, ranges = x.ranges, score_stride = x.score_stride, max_kv_len = x.max_kv_len, n_pages = x.n_pages,
              n_seqs = x.n_seqs, max_q_len = x.max_q_len, nh = x.nh, nkv = x.nkv, hd = x.hd;
    const float scale = x.scale;
    if (n_seqs == 0 || max_q_len == 0) return 0;
    int rc = c8_check("attention8", x.codes, x.scales, page_size, n_pages, nkv, hd, x.table_stride);
    if (!rc) rc = check_step("attention8", nh, nkv, n_seqs, max_q_len, window);
    if (rc) return rc;
    TQ_REQUIRE(ranges >= 1 && ranges <= (partial != nullptr ? JOIN_RANGES : CLUSTER), "attention8: %d ranges need a buffer for their sums", ranges);
    TQ_REQUIRE((scores == nullptr) == (weights == nullptr) && (scores == nullptr || (max_q_len == 1 && (partial != nullptr || ranges > 1) && score_stride >= max_kv_len && (uintptr_t)scores % 16 == 0)),
               "attention8: scores of %d places do not hold %d", score_stride, max_kv_len);
    const Cache8 c = c8_cache(x.codes, x.scales, x.page_table, x.table_stride, page_size, n_pages, nkv, hd);
    const Step S{x.cu_seqlens, x.held, nh, window, scale * LOG2E};
    const int columns = max_q_len * (nh / nkv);
    auto first = [&]() -> int {
        TQ_DISPATCH(x.act_dtype, TA,
#define C8_CALL(HDP, NT, EXACT) (launch8<Form<TA, HDP, NT, EXACT>>(q, c, S, x.out, partial, ranges, scores, score_stride, partial == nullptr ? x.lse : nullptr, partial == nullptr ? weights : nullptr, n_seqs, max_q_len, x.stream))
            C8_FORMS(columns, C8_CALL));
#undef C8_CALL
        return -2;
    };
    rc = first();
    if (rc || partial == nullptr) return rc;
    const int chunks = weights != nullptr ? (max_kv_len + 127) / 128 : 0;
    TQ_DISPATCH(x.act_dtype, TA, tq_launch(dim3(columns + chunks, nkv, n_seqs), 128, 0, x.stream)(join8_kernel<TA>, c, S, partial, ranges, (TA*)x.out, columns, x.lse, scores, score_stride, weights));
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
    const Cache8 c = c8_cache(codes, scales, page_table, table_stride, page_size, n_pages, nkv, hd);
    const Step S{cu_seqlens, held, nh, window, scale * LOG2E};
    return hd == 64 ? launch_repair8<Form<__nv_bfloat16, 64, 2, true>>(q, c, S, out, lost, lost_stride, n_seqs, stream) : launch_repair8<Form<__nv_bfloat16, 128, 2, true>>(q, c, S, out, lost, lost_stride, n_seqs, stream);
}

// weights of places below held[s] grow by, those of the step's own rows become, the sum over the step's rows and the head's query heads of
// 2^(score - lse).  max_kv_len: at least the longest held[s] + run.
TQ_EXPORT int tq_weigh8(const void* q, const void* codes, const void* scales, int act_dtype, const int* cu_seqlens, const int* held,
                        const int* page_table, int table_stride, int page_size, int window, float scale, const float* lse, float* weights, int n_pages,
                        int n_seqs, int max_kv_len, int nh, int nkv, int hd, cudaStream_t stream) {
    if (n_seqs == 0 || max_kv_len == 0) return 0;
    int rc = c8_check("weigh8", codes, scales, page_size, n_pages, nkv, hd, table_stride);
    if (!rc) rc = check_step("weigh8", nh, nkv, n_seqs, max_kv_len, window);
    if (rc) return rc;
    const Cache8 c = c8_cache(codes, scales, page_table, table_stride, page_size, n_pages, nkv, hd);
    const Step S{cu_seqlens, held, nh, window, scale * LOG2E};
    TQ_DISPATCH(act_dtype, TA,
        if (hd <= 64) return launch_weigh8<Form<TA, 64, 1, false>, 4>(q, c, S, lse, weights, n_seqs, max_kv_len, stream);
        if (hd <= 128) return launch_weigh8<Form<TA, 128, 1, false>, 4>(q, c, S, lse, weights, n_seqs, max_kv_len, stream);
        return launch_weigh8<Form<TA, 256, 1, false>, 2>(q, c, S, lse, weights, n_seqs, max_kv_len, stream));
    return -2;
}
