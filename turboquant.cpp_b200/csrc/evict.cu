// Eviction from the 8-bit cache (layout and codes: cache8.cuh): sequences that hold more rows than a budget keep, in every key/value head,
// the newest `recent` ones and, of the others, those whose accumulated attention weight is largest.
//
//   tq_evict8   two launches: which rows stay, per sequence and key/value head a list of places, ascending; then the rows of the lists, their
//               bytes and their sums of weights, to new pages
#include "cache8.cuh"

TQ_DEFINE_LAST_ERROR

namespace {

// Floats in an order that unsigned integers have, NaN (either sign) below everything, both zeros equal.
__device__ __forceinline__ uint32_t rank_of(float w) {
    if (w != w) return 0u;
    const uint32_t u = __float_as_uint(w + 0.0f);                     // -0 + 0 = +0
    return (u & 0x80000000u) ? ~u : u | 0x80000000u;
}

// ---------------------------------------------------------------------------------------
// Selection: a block per (key/value head, sequence) finds the rank of the last row that stays, 11 bits at a time from the highest in which the
// ranks differ at all (a histogram of the rows that agree in the bits found; once a bin holds few rows they are compared one by one), then
// lists the rows above it and, of those equal to it, the first ones.  Ranks are counted from the smallest one, so that the first histogram
// spreads over its bins: with the 11 highest bits of the float a handful of bins took all rows, and the additions to them queued.  A thread
// takes four consecutive rows of a page, one load of it and one of the page table; the ranks stay in shared memory as far as they fit (`cached` of them).
// 32 sequences of about 7,000 rows, 4 heads: 9 us, of them 2 for the reads, 5 for the histograms, 2 for the lists: latencies of one block an SM
// (row by row, bits from the top: 14.6).  Where a row a thread covers a sequence that is shorter (960 rows of 16 heads, with the moving: 8.8 us, by
// fours 10.3; 1,600 rows 8.9 and 8.4).
// ---------------------------------------------------------------------------------------
constexpr int SELECT_THREADS = 1024, SELECT_WARPS = SELECT_THREADS / 32, DIGIT = 11, BINS = 1 << DIGIT;
constexpr int FEW = 64;                 // rows of a bin that are told apart one by one
constexpr int SELECT_MOST = 48 * 1024;             // ranks a block keeps, 192 KB

template <int PER>
__global__ void __launch_bounds__(SELECT_THREADS) evict8_select_kernel(Cache8 c, const float* __restrict__ weights, const int* __restrict__ lengths, int budget, int recent,
                                                                       int cached, int* __restrict__ kept) {
    tq_grid_wait();                    // everything below may read what the previous kernel wrote
    tq_grid_launch_dependents();
    constexpr int ROUND = PER * SELECT_THREADS;        // rows the block looks at at once
    extern __shared__ __align__(16) uint32_t s_rank[];
    __shared__ uint32_t s_few[FEW];
    __shared__ int s_hist[BINS], s_pick[4], s_warp[2][SELECT_WARPS], s_own[SELECT_WARPS];
    const int g = blockIdx.x, seq = blockIdx.y, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int n = max(0, min(lengths[seq], c.table_stride * c.page_size));
    int* list = kept + ((size_t)seq * c.nkv + g) * budget;
    if (n <= budget) {
        for (int j = tid; j < budget; j += SELECT_THREADS) list[j] = j < n ? j : -1;
        return;
    }
    const int rest = n - recent, want = budget - recent;              // of places 0 .. rest - 1 `want` stay
    for (int j = tid; j < recent; j += SELECT_THREADS) list[want + j] = rest + j;
    if (want == 0) return;
    // the ranks of places p .. p + PER - 1: one page has all of them
    struct alignas(4 * PER) Ranks { uint32_t k[PER]; };
    auto read = [&](int p) {
        const float* w = weights + ((size_t)c.page_of(seq, p) * c.nkv + g) * c.page_size + c.row(p);
        Ranks f;
        if constexpr (PER == 4) {
            const float4 v = *reinterpret_cast<const float4*>(w);
            f = {{rank_of(v.x), rank_of(v.y), rank_of(v.z), rank_of(v.w)}};
        } else f = {{rank_of(*w)}};
        return f;
    };
    auto ranks = [&](int p) { return p >= rest ? Ranks{} : p < cached ? *reinterpret_cast<const Ranks*>(s_rank + p) : read(p); };
    uint32_t least = 0xffffffffu, most = 0u;
    for (int p = PER * tid; p < rest; p += ROUND) {
        const Ranks f = read(p);
        if (p < cached) *reinterpret_cast<Ranks*>(s_rank + p) = f;
#pragma unroll
        for (int i = 0; i < PER; ++i)
            if (p + i < rest) { least = min(least, f.k[i]); most = max(most, f.k[i]); }
    }
    least = __reduce_min_sync(0xffffffffu, least);
    most = __reduce_max_sync(0xffffffffu, most);
    if (lane == 0) { s_warp[0][warp] = (int)least; s_warp[1][warp] = (int)most; }
    __syncthreads();
    least = __reduce_min_sync(0xffffffffu, (uint32_t)s_warp[0][lane]);
    most = __reduce_max_sync(0xffffffffu, (uint32_t)s_warp[1][lane]);
    uint32_t found = 0;                                               // the rank of the last row that stays, less `least`: its highest bits
    int missing = want;                                               // rows still to be found among those that agree with them
    for (int left = 32 - __clz(most - least); left > 0;) {            // bits not yet found
        const int shift = max(left - DIGIT, 0);
        *reinterpret_cast<int2*>(s_hist + 2 * tid) = make_int2(0, 0);
        __syncthreads();
        for (int p0 = 0; p0 < rest; p0 += ROUND) {
            const int p = p0 + PER * tid;
            const Ranks f = ranks(p);
            uint32_t d[PER];
            bool counts[PER], any = false;
#pragma unroll
            for (int i = 0; i < PER; ++i) {
                d[i] = (f.k[i] - least) ^ found;                      // found: no bits below `left`
                counts[i] = p + i < rest && (left == 32 || d[i] >> left == 0);
                any |= counts[i];
            }
            if (!__any_sync(0xffffffffu, any)) continue;
#pragma unroll
            for (int i = 0; i < PER; ++i) {
                const uint32_t lanes = __ballot_sync(0xffffffffu, counts[i]);
                if (lanes == 0) continue;
                // one lane's bin is counted once for all lanes that share it (rows that never received any weight are many)
                const int bin = counts[i] ? (int)(d[i] >> shift) : -1, leader = __ffs(lanes) - 1, lead = __shfl_sync(0xffffffffu, bin, leader);
                const uint32_t same = __ballot_sync(0xffffffffu, bin == lead);
                if (lane == leader) atomicAdd(&s_hist[lead], __popc(same));
                if (counts[i] && bin != lead) atomicAdd(&s_hist[bin], 1);
            }
        }
        __syncthreads();
        // a thread has two bins, thread 0 the highest: rows in them and, scanned over the block, in those above
        const int high = BINS - 1 - 2 * tid, in_high = s_hist[high], sum = in_high + s_hist[high - 1];
        int above = sum;
        for (int o = 1; o < 32; o <<= 1) {
            const int v = __shfl_up_sync(0xffffffffu, above, o);
            if (lane >= o) above += v;
        }
        if (lane == 31) s_warp[0][warp] = above;
        __syncthreads();
        above += __reduce_add_sync(0xffffffffu, lane < warp ? s_warp[0][lane] : 0);
        const int before = above - sum;
        if (before < missing && missing <= above) {
            const bool first = missing - before <= in_high;
            s_pick[0] = first ? high : high - 1;
            s_pick[1] = missing - before - (first ? 0 : in_high);
            s_pick[2] = first ? in_high : sum - in_high;
            s_pick[3] = 0;
        }
        __syncthreads();
        found |= (uint32_t)s_pick[0] << shift;
        missing = s_pick[1];
        left = shift;
        if (missing == s_pick[2]) {                                   // all rows of the bin stay: those above `found` - 1 (it is not the lowest, or all of `rest` would stay)
            found -= 1;
            missing = 0;
            break;
        }
        if (left > 0 && s_pick[2] <= FEW) {                           // the bin's rows, each compared to all
            const int few = s_pick[2];
            for (int p = PER * tid; p < rest; p += ROUND) {
                const Ranks f = ranks(p);
#pragma unroll
                for (int i = 0; i < PER; ++i) {
                    const uint32_t d = f.k[i] - least;
                    if (p + i < rest && (d ^ found) >> left == 0) s_few[atomicAdd(&s_pick[3], 1)] = d;
                }
            }
            __syncthreads();
            if (tid < few) {
                const uint32_t d = s_few[tid];
                int higher = 0, equal = 0;
                for (int i = 0; i < few; ++i) { higher += s_few[i] > d; equal += s_few[i] == d; }
                if (higher < missing && missing <= higher + equal) { s_pick[0] = (int)d; s_pick[1] = missing - higher; }       // (rows of one rank write alike)
            }
            __syncthreads();
            found = (uint32_t)s_pick[0];
            missing = s_pick[1];
            break;
        }
    }
    const uint32_t last = least + found;
    // rows above `last` stay, and the first `missing` of those equal to it: a scan over the block of how many of each a thread has, 16 bits each
    int a = 0, e = 0;                                                 // those of the rounds before
    for (int p0 = 0; p0 < rest; p0 += ROUND) {
        const int p = p0 + PER * tid;
        const Ranks f = ranks(p);
        int own = 0;
#pragma unroll
        for (int i = 0; i < PER; ++i)
            if (p + i < rest) own += f.k[i] > last ? 1 << 16 : f.k[i] == last ? 1 : 0;
        int upto = own;
        for (int o = 1; o < 32; o <<= 1) {
            const int v = __shfl_up_sync(0xffffffffu, upto, o);
            if (lane >= o) upto += v;
        }
        if (lane == 31) s_own[warp] = upto;
        __syncthreads();
        const int of_warp = s_own[lane], before = __reduce_add_sync(0xffffffffu, lane < warp ? of_warp : 0) + upto - own;
        int a1 = a + (before >> 16), e1 = e + (before & 0xffff);
#pragma unroll
        for (int i = 0; i < PER; ++i) {
            if (p + i >= rest) break;
            if (f.k[i] > last) list[a1++ + min(e1, missing)] = p + i;
            else if (f.k[i] == last && e1++ < missing) list[a1 + e1 - 1] = p + i;
        }
        const int all = __reduce_add_sync(0xffffffffu, of_warp);
        a += all >> 16;
        e += all & 0xffff;
        __syncthreads();
    }
}

// ---------------------------------------------------------------------------------------
// Moving: a warp per 16 rows of the list, a lane for each row and plane on the way to its page and byte.  The new block's byte is the largest of
// its rows' bytes; rows of a smaller one are rounded again.  Nothing is shared between warps.  2,048 of about 7,000 rows of 32 sequences, 4 heads of 128:
// 32 us for 134 MB, about the time of reading all of the old pages: 128 bytes in three of every 384.  (A warp per 64 rows and plane, which goes
// that way once for four times as many, was slower by a fifth: too few warps;
// so was a warp that looked up two or four blocks' rows at once.  Rows that lie side by side take 24 us.)
// ---------------------------------------------------------------------------------------
// HD: the head size, or 0 where it is known at the launch only (then a division for each piece: 36 us for the rows above).
template <int HD>
__global__ void __launch_bounds__(256) evict8_move_kernel(Cache8 c, float* __restrict__ weights, const int* __restrict__ kept, const int* __restrict__ new_table,
                                                          int new_stride, int budget) {
    tq_grid_wait();                    // everything below may read what the previous kernel wrote
    tq_grid_launch_dependents();
    const int lane = threadIdx.x & 31, plane = lane >> 4, r = lane & 15, first = (blockIdx.x * 8 + (threadIdx.x >> 5)) * C8_BLOCK, seq = blockIdx.z, g = blockIdx.y;
    if (first >= budget) return;
    const int* list = kept + ((size_t)seq * c.nkv + g) * budget;
    const int place = first + r < budget ? list[first + r] : -1;
    const int listed = new_table[(size_t)seq * new_stride + TQ_CHECKED(c.column(first), new_stride, TQ_IDX_TABLE_COLUMN)];
    const int rows = __popc(__ballot_sync(0xffffffffu, place >= 0) & 0xffffu), row0 = c.row(first), hd = HD ? HD : c.hd, vecs = hd / 16;
    if (rows == 0) return;                                            // the list ends before these: they need no page
    const int page = TQ_CHECKED(listed, c.n_pages, TQ_IDX_PAGE);
    unsigned long long from = 0;
    uint32_t byte = 0;
    float weight = 0.f;
    if (place >= 0) {
        const int old = c.page_of(seq, place), row = c.row(place);
        from = c.codes_at(old, plane, g) + (size_t)row * hd;
        byte = c.scales[c.scales_at(old, plane, g) + row / C8_BLOCK];
        if (plane == 0) weight = weights[((size_t)old * c.nkv + g) * c.page_size + row];
    }
    const size_t to = c.codes_at(page, 0, g) + (size_t)row0 * hd, between = (size_t)c.nkv * c.page_size * hd;
    uint32_t top = byte;
#pragma unroll
    for (int o = 8; o > 0; o >>= 1) top = max(top, __shfl_xor_sync(0xffffffffu, top, o));
    const uint32_t shift = top - byte;
    // pieces of 16 bytes: all rows of the keys, then of the values
    const int pieces = C8_BLOCK * vecs;
    constexpr int BATCH = 8;               // all of them asked for before the first is stored (the compiler cannot know that they do not overlap)
    for (int v0 = 0; v0 < 2 * pieces; v0 += 32 * BATCH) {
        uint4 x[BATCH];
#pragma unroll
        for (int i = 0; i < BATCH; ++i) {
            const int v = v0 + 32 * i + lane, which = v / vecs, at = (v - which * vecs) * 16;        // which: row, 16 more for values
            const unsigned long long src = __shfl_sync(0xffffffffu, from, which & 31);
            if (v < 2 * pieces && (which & 15) < rows) x[i] = *reinterpret_cast<const uint4*>(c.codes + src + at);
        }
#pragma unroll
        for (int i = 0; i < BATCH; ++i) {
            const int v = v0 + 32 * i + lane, which = v / vecs, at = (v - which * vecs) * 16;
            const uint32_t s = __shfl_sync(0xffffffffu, shift, which & 31);
            if (v < 2 * pieces && (which & 15) < rows) {
                if (s) x[i] = c8_shift16(x[i], c8_shift_factor((int)min(s, 25u)));
                *reinterpret_cast<uint4*>(c.codes + to + (which >> 4) * between + (size_t)(which & 15) * hd + at) = x[i];
            }
        }
    }
    if (r == 0) c.scales[c.scales_at(page, plane, g) + row0 / C8_BLOCK] = (uint8_t)top;
    if (plane == 0 && place >= 0) weights[((size_t)page * c.nkv + g) * c.page_size + row0 + r] = weight;
}

}  // namespace

// lengths [n_seqs] (device): rows each sequence holds; kept [n_seqs, nkv, budget]: receives the places that stay, ascending, then -1.  Row j of
// them goes to place j of new_table's pages, none of which holds any of these rows.
struct Evict8Call {
    void *codes, *scales;
    float* weights;
    const int *lengths, *page_table, *new_table;
    int* kept;
    cudaStream_t stream;
    int table_stride, new_stride, page_size, n_pages, n_seqs, nkv, hd, budget, recent;
};
TQ_EXPORT int tq_evict8(const void* packed, int bytes) {
    C8_REQUIRE_CALL("evict8", Evict8Call);
    const Evict8Call x = c8_call<Evict8Call>(packed);
    const int* page_table = x.page_table;
    const int table_stride = x.table_stride, page_size = x.page_size, n_pages = x.n_pages, n_seqs = x.n_seqs, nkv = x.nkv, hd = x.hd, budget = x.budget, recent = x.recent;
    if (n_seqs == 0) return 0;
    int rc = c8_check("evict8", x.codes, x.scales, page_size, n_pages, nkv, hd, table_stride);
    if (rc) return rc;
    TQ_REQUIRE(budget >= 1 && recent >= 0 && recent <= budget, "evict8: %d newest of a budget of %d rows", recent, budget);
    TQ_REQUIRE((long long)x.new_stride * page_size >= budget, "evict8: %d new pages a sequence for a budget of %d rows", x.new_stride, budget);
    TQ_REQUIRE(n_seqs <= 65535 && nkv <= 65535, "evict8: %d sequences, %d heads", n_seqs, nkv);
    TQ_REQUIRE((long long)table_stride * page_size < (1ll << 31), "evict8: page tables of %d pages", table_stride);
    TQ_REQUIRE(x.weights != nullptr && (uintptr_t)x.weights % 16 == 0, "evict8: weights must be there, and 16-byte aligned");
    const Cache8 c = c8_cache(x.codes, x.scales, page_table, table_stride, page_size, n_pages, nkv, hd);
    const int cached = table_stride * page_size < SELECT_MOST ? table_stride * page_size : SELECT_MOST;
    const bool small = table_stride * page_size - recent <= SELECT_THREADS;
    static TqSmemAsked asked[2];
    const auto select = small ? evict8_select_kernel<1> : evict8_select_kernel<4>;
    const cudaError_t e = tq_grow_smem(select, (size_t)cached * 4, asked[small]);
    if (e != cudaSuccess) TQ_FAIL(-1, "evict8: cannot reserve %d bytes of shared memory: %s", cached * 4, cudaGetErrorString(e));
    tq_launch(dim3(nkv, n_seqs), SELECT_THREADS, (size_t)cached * 4, x.stream)(select, c, x.weights, x.lengths, budget, recent, cached, x.kept);
    TQ_CHECK_LAUNCH("evict8_select");
    const auto move = hd == 128 ? evict8_move_kernel<128> : hd == 64 ? evict8_move_kernel<64> : evict8_move_kernel<0>;
    tq_launch(dim3(((budget + C8_BLOCK - 1) / C8_BLOCK + 7) / 8, nkv, n_seqs), 256, 0, x.stream)(move, c, x.weights, x.kept, x.new_table, x.new_stride, budget);
    TQ_CHECK_LAUNCH("evict8_move");
    return 0;
}
