// Eviction from the 8-bit cache (layout and codes: cache8.cuh): sequences that hold more rows than a budget keep, in every key/value head,
// the newest `recent` ones and, of the others, those whose accumulated attention weight is largest.
//
//   tq_evict8_select   which rows stay: per sequence and key/value head a list of places, ascending
//   tq_evict8_move     the rows of such a list, their bytes and their sums of weights, to new pages
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
// Selection: a block per (key/value head, sequence) finds the rank of the last row that stays, a byte at a time from the highest (a
// histogram of the rows that agree in the bytes found), then lists the rows above it and, of those equal to it, the first ones.
// ---------------------------------------------------------------------------------------
constexpr int SELECT_THREADS = 1024;

__global__ void __launch_bounds__(SELECT_THREADS) evict8_select_kernel(const float* __restrict__ weights, const int* __restrict__ lengths, const int* __restrict__ table,
                                                                       int table_stride, int page_size, int n_pages, int nkv, int budget, int recent, int* __restrict__ kept) {
    tq_grid_wait();                    // everything below may read what the previous kernel wrote
    tq_grid_launch_dependents();
    __shared__ int s_hist[256], s_pick[2], s_sum[2][SELECT_THREADS / 32];
    const int g = blockIdx.x, seq = blockIdx.y, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int n = max(0, min(lengths[seq], table_stride * page_size));
    int* list = kept + ((size_t)seq * nkv + g) * budget;
    if (n <= budget) {
        for (int j = tid; j < budget; j += SELECT_THREADS) list[j] = j < n ? j : -1;
        return;
    }
    const int rest = n - recent, want = budget - recent;              // of places 0 .. rest - 1 `want` stay
    for (int j = tid; j < recent; j += SELECT_THREADS) list[want + j] = rest + j;
    if (want == 0) return;
    const int* pages = table + (size_t)seq * table_stride;
    auto rank_at = [&](int p) {
        const int page = TQ_CHECKED(pages[p / page_size], n_pages, TQ_IDX_PAGE);
        return rank_of(weights[((size_t)page * nkv + g) * page_size + p % page_size]);
    };
    uint32_t prefix = 0;
    int missing = want;                                               // rows still to be found among those that agree with the prefix
    for (int shift = 24; shift >= 0; shift -= 8) {
        if (tid < 256) s_hist[tid] = 0;
        __syncthreads();
        for (int p = tid; p < rest; p += SELECT_THREADS) {
            const uint32_t k = rank_at(p);
            if (shift == 24 || (k >> (shift + 8)) == (prefix >> (shift + 8))) atomicAdd(&s_hist[(k >> shift) & 255u], 1);
        }
        __syncthreads();
        if (warp == 0) {                                              // lane i: bins 255 - 8 i downwards
            int sum = 0;
            for (int j = 0; j < 8; ++j) sum += s_hist[255 - 8 * lane - j];
            int above = sum;                                          // rows in the bins of this lane and those before it
            for (int o = 1; o < 32; o <<= 1) {
                const int v = __shfl_up_sync(0xffffffffu, above, o);
                if (lane >= o) above += v;
            }
            const int before = above - sum;
            if (before < missing && missing <= above) {
                int left = missing - before, bin = 255 - 8 * lane;
                while (s_hist[bin] < left) left -= s_hist[bin--];
                s_pick[0] = bin;
                s_pick[1] = left;
            }
        }
        __syncthreads();
        prefix |= (uint32_t)s_pick[0] << shift;
        missing = s_pick[1];
        __syncthreads();
    }
    // rows above `prefix` stay, and the first `missing` of those equal to it
    int base_above = 0, base_equal = 0;
    for (int p0 = 0; p0 < rest; p0 += SELECT_THREADS) {
        const int p = p0 + tid;
        const uint32_t k = p < rest ? rank_at(p) : 0u;
        const bool above = p < rest && k > prefix, equal = p < rest && k == prefix;
        const uint32_t am = __ballot_sync(0xffffffffu, above), em = __ballot_sync(0xffffffffu, equal), below = (1u << lane) - 1u;
        if (lane == 0) { s_sum[0][warp] = __popc(am); s_sum[1][warp] = __popc(em); }
        __syncthreads();
        int a = base_above + __popc(am & below), e = base_equal + __popc(em & below);
        for (int w = 0; w < SELECT_THREADS / 32; ++w) {
            if (w < warp) { a += s_sum[0][w]; e += s_sum[1][w]; }
            base_above += s_sum[0][w];
            base_equal += s_sum[1][w];
        }
        if (above || (equal && e < missing)) list[a + min(e, missing)] = p;
        __syncthreads();
    }
}

// ---------------------------------------------------------------------------------------
// Moving: a block per 16 rows of the list.  The new block's byte is the largest of its rows' bytes; rows of a smaller one are rounded again.
// ---------------------------------------------------------------------------------------
__global__ void __launch_bounds__(128) evict8_move_kernel(Cache8 c, float* __restrict__ weights, const int* __restrict__ kept, const int* __restrict__ new_table,
                                                          int new_stride, int budget) {
    tq_grid_wait();                    // everything below may read what the previous kernel wrote
    tq_grid_launch_dependents();
    __shared__ size_t s_from[2][C8_BLOCK];
    __shared__ uint32_t s_byte[2][C8_BLOCK];
    const int seq = blockIdx.z, g = blockIdx.y, first = blockIdx.x * C8_BLOCK, tid = threadIdx.x;
    const int* list = kept + ((size_t)seq * c.nkv + g) * budget;
    const int rows = min(C8_BLOCK, budget - first);
    if (list[first] < 0) return;                                      // the list ends before this block
    const int page = TQ_CHECKED(new_table[(size_t)seq * new_stride + TQ_CHECKED(first / c.page_size, new_stride, TQ_IDX_TABLE_COLUMN)], c.n_pages, TQ_IDX_PAGE);
    const int row0 = first % c.page_size;
    if (tid < 2 * C8_BLOCK) {
        const int plane = tid / C8_BLOCK, r = tid % C8_BLOCK, place = r < rows ? list[first + r] : -1;
        uint32_t byte = 0;
        if (place >= 0) {
            const int from = c.page_of(seq, place), row = place % c.page_size;
            byte = c.scales[c.scales_at(from, plane, g) + row / C8_BLOCK];
            s_from[plane][r] = c.codes_at(from, plane, g) + (size_t)row * c.hd;
            if (plane == 0) weights[((size_t)page * c.nkv + g) * c.page_size + row0 + r] = weights[((size_t)from * c.nkv + g) * c.page_size + row];
        }
        uint32_t top = byte;
        for (int o = 8; o > 0; o >>= 1) top = max(top, __shfl_xor_sync(0xffffffffu, top, o));
        s_byte[plane][r] = place < 0 ? 256u : top - byte;             // how far the row's codes move; 256: no row
        if (r == 0) c.scales[c.scales_at(page, plane, g) + row0 / C8_BLOCK] = (uint8_t)top;
    }
    __syncthreads();
    const int vecs = c.hd / 16;
    for (int v = tid; v < 2 * C8_BLOCK * vecs; v += blockDim.x) {
        const int plane = v / (C8_BLOCK * vecs), r = v / vecs % C8_BLOCK, at = v % vecs;
        const uint32_t shift = s_byte[plane][r];
        if (shift == 256u) continue;
        uint4 x = *reinterpret_cast<const uint4*>(c.codes + s_from[plane][r] + at * 16);
        if (shift) x = c8_shift16(x, c8_shift_factor((int)min(shift, 25u)));
        *reinterpret_cast<uint4*>(c.codes + c.codes_at(page, plane, g) + (size_t)(row0 + r) * c.hd + at * 16) = x;
    }
}

}  // namespace

// lengths [n_seqs] (device): rows each sequence holds; kept [n_seqs, nkv, budget]: the places that stay, ascending, then -1.
TQ_EXPORT int tq_evict8_select(const float* weights, const int* lengths, const int* page_table, int table_stride, int page_size, int n_pages, int n_seqs,
                               int nkv, int budget, int recent, int* kept, cudaStream_t stream) {
    if (n_seqs == 0) return 0;
    TQ_REQUIRE(budget >= 1 && recent >= 0 && recent <= budget, "evict8: %d newest of a budget of %d rows", recent, budget);
    TQ_REQUIRE(page_size >= 1 && table_stride >= 1 && nkv >= 1 && n_seqs <= 65535, "evict8: page size %d, tables %d wide, %d heads, %d sequences", page_size, table_stride, nkv, n_seqs);
    TQ_REQUIRE((long long)table_stride * page_size < (1ll << 31), "evict8: page tables of %d pages", table_stride);
    tq_launch(dim3(nkv, n_seqs), SELECT_THREADS, 0, stream)(evict8_select_kernel, weights, lengths, page_table, table_stride, page_size, n_pages, nkv, budget, recent, kept);
    TQ_CHECK_LAUNCH("evict8_select");
    return 0;
}

// The rows that `kept` lists, row j to place j of new_table's pages, which hold none of the listed rows.
TQ_EXPORT int tq_evict8_move(void* codes, void* scales, float* weights, const int* kept, const int* page_table, int table_stride, const int* new_table,
                             int new_stride, int page_size, int n_pages, int n_seqs, int nkv, int hd, int budget, cudaStream_t stream) {
    if (n_seqs == 0) return 0;
    int rc = c8_check("evict8", codes, scales, page_size, n_pages, nkv, hd, table_stride);
    if (rc) return rc;
    TQ_REQUIRE(budget >= 1 && (long long)new_stride * page_size >= budget, "evict8: %d new pages a sequence for a budget of %d rows", new_stride, budget);
    TQ_REQUIRE(n_seqs <= 65535 && nkv <= 65535, "evict8: %d sequences, %d heads", n_seqs, nkv);
    const Cache8 c{(uint8_t*)codes, (uint8_t*)scales, page_table, table_stride, page_size, n_pages, nkv, hd};
    tq_launch(dim3((budget + C8_BLOCK - 1) / C8_BLOCK, nkv, n_seqs), 128, 0, stream)(evict8_move_kernel, c, weights, kept, new_table, new_stride, budget);
    TQ_CHECK_LAUNCH("evict8_move");
    return 0;
}
