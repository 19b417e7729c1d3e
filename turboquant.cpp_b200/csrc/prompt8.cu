// Prompts over the 8-bit cache (layout and codes: cache8.cuh).
//
//   tq_expand8         the pages a step sees as bfloat16 pages of a scratch cache, which the tensor-core prompt kernel then reads
//   tq_weigh8_prompt   sums of softmax weights over a prompt's rows, from the same scratch, on the tensor cores
#include "cache8.cuh"
#include "umma.cuh"

TQ_DEFINE_LAST_ERROR

namespace {

constexpr int PAGE = 64;

// ---------------------------------------------------------------------------------------
// A page of one key/value head, both planes.  e4m3 times a power of two is a bfloat16 value: nothing is rounded (below 2^-133 apart).  Rows
// behind the sequence's last become zeros, since the prompt kernel reads whole pages; pages that hold a NaN among the values are marked.
// Bound by memory: 12,000 rows of 16 heads of 128, 49 MB in and 98 MB out, some 20 us of the prompt's 168.
// ---------------------------------------------------------------------------------------
__device__ __forceinline__ uint32_t bf16x2_of(uint32_t two, float scale) {
    const uint32_t h = c8_half2(two);
    float lo, hi;
    asm("{\n\t.reg .b16 l, h;\n\tmov.b32 {l, h}, %2;\n\tcvt.f32.f16 %0, l;\n\tcvt.f32.f16 %1, h;\n\t}" : "=f"(lo), "=f"(hi) : "r"(h));
    const __nv_bfloat162 b = __floats2bfloat162_rn(lo * scale, hi * scale);
    return *reinterpret_cast<const uint32_t*>(&b);
}

// the first page of a sequence that a step's rows see
__device__ __forceinline__ int first_page(int start, int window) { return (window > 0 ? max(0, start + 1 - window) : 0) / PAGE; }

__global__ void __launch_bounds__(256) expand8_kernel(Cache8 c, const int* __restrict__ cu_seqlens, const int* __restrict__ held, int window, uint4* __restrict__ dense,
                                                      int* __restrict__ dense_table, uint8_t* __restrict__ lost, int width, int dense_width) {
    tq_grid_wait();                    // everything below may read what the previous kernel wrote
    tq_grid_launch_dependents();
    const int n = blockIdx.x, g = blockIdx.y, seq = blockIdx.z, start = held[seq], run = cu_seqlens[seq + 1] - cu_seqlens[seq], last = start + run - 1;
    const int first = first_page(start, window);
    if (run <= 0 || n * PAGE > last || n < first || n - first >= dense_width) return;
    const int page = c.page_of(seq, n * PAGE), to = seq * dense_width + n - first, vecs = c.hd / 16, rows = min(PAGE, last + 1 - n * PAGE);
    bool nan = false;
    const uint8_t* codes = c.codes + c.codes_at(page, 0, g);
    const uint8_t* scales = c.scales + c.scales_at(page, 0, g);
    const size_t plane_codes = (size_t)c.nkv * PAGE * c.hd, plane_scales = (size_t)c.nkv * (PAGE / C8_BLOCK);
    constexpr int BATCH = 4;                   // pieces of 16 codes a thread asks for at a time
    const int pieces = PAGE * vecs;
    for (int i0 = threadIdx.x; i0 < 2 * pieces; i0 += 256 * BATCH) {
        uint4 x[BATCH];
        float s[BATCH];
#pragma unroll
        for (int k = 0; k < BATCH; ++k) {
            const int i = i0 + 256 * k, plane = i >= pieces, j = i - plane * pieces, r = j / vecs;
            x[k] = make_uint4(0, 0, 0, 0);
            s[k] = 1.f;
            if (i < 2 * pieces && r < rows) {
                x[k] = __ldcg(reinterpret_cast<const uint4*>(codes + plane * plane_codes) + j);
                s[k] = c8_scale(__ldcg(scales + plane * plane_scales + r / C8_BLOCK));
            }
        }
#pragma unroll
        for (int k = 0; k < BATCH; ++k) {
            const int i = i0 + 256 * k, plane = i >= pieces, j = i - plane * pieces;
            if (i >= 2 * pieces) break;
            const uint32_t u[4] = {x[k].x, x[k].y, x[k].z, x[k].w};
            uint32_t w[8];
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                w[2 * e] = bf16x2_of(u[e] & 0xffffu, s[k]);
                w[2 * e + 1] = bf16x2_of(u[e] >> 16, s[k]);
                nan |= plane == 1 && (((u[e] & 0x7f7f7f7fu) + 0x01010101u) & 0x80808080u) != 0;
            }
            uint4* d = dense + (((size_t)to * 2 + plane) * c.nkv + g) * (pieces * 2) + (size_t)j * 2;
            d[0] = make_uint4(w[0], w[1], w[2], w[3]);
            d[1] = make_uint4(w[4], w[5], w[6], w[7]);
        }
    }
    const bool any = __syncthreads_or(nan);
    if (threadIdx.x == 0) {
        lost[((size_t)seq * c.nkv + g) * width + n] = any ? 1 : 0;
        if (g == 0) dense_table[seq * width + n] = to;
    }
}

// ---------------------------------------------------------------------------------------
// Sums of weights of a prompt: with the rows' denominators known, sum over rows and heads of 2^(factor q.k - lse) needs one product and no
// running maximum.  A CTA keeps 128 keys of one key/value head as the left operand and lets the query tiles that see them pass, so that a
// thread holds one key's scores against 128 rows and adds them up in its own register: no reduction, no atomics, one writer per sum and a
// fixed order.  Two accumulators in tensor memory, one for each of two groups of four warps: one group's exponentials (the bound: 16,384 a
// tile at 16 a cycle and SM) run beside the other's product.  Two CTAs share an SM.  A prompt of 2,048 rows, 16 heads of 128: 18 us (the CTA
// of the first keys walks 16 tiles, the last one's one), where the same sums on mma.sync, each query tile converted for 64 keys, took 650.
//   warp 0   TMA: the keys once, then query tiles through a ring      warp 1   owns tensor memory, issues S = K Q^T
//   warps 2..5 and 6..9   every other tile each
// ---------------------------------------------------------------------------------------
template <int DK> struct WCfg {
    static constexpr int KB = DK / 64, TILE = BM * DK * 2, PAGE_BYTES = PAGE * DK * 2, STAGES = 2;
    static constexpr int SMEM_BYTES = (1 + STAGES) * TILE + 1024;
};
constexpr int W_THREADS = 320;

struct WShape { int nh, nkv, width, window, table_stride, n_pages; float factor; };

template <int DK>
__global__ void __launch_bounds__(W_THREADS, 2)
weigh8_prompt_kernel(const __grid_constant__ CUtensorMap map_q, const __grid_constant__ CUtensorMap map_k, const __grid_constant__ WShape S,
                     const int* __restrict__ cu_seqlens, const int* __restrict__ held, const int* __restrict__ page_table, const float* __restrict__ lse,
                     float* __restrict__ weights, int* __restrict__ status) {
    tq_grid_wait();                    // everything below may read what the previous kernel wrote
    using C = WCfg<DK>;
    extern __shared__ uint8_t smem_raw[];
    __shared__ int s_abort;
    __shared__ uint32_t s_tmem_base;
    __shared__ __align__(8) uint64_t s_bars[1 + 2 * C::STAGES + 4];
    __shared__ __align__(16) float s_lse[8][BM];           // a warp's own copy of its tile's denominators: no barrier that an abort could leave waiting
    __shared__ float s_sum[2][BM];
    const int g = blockIdx.x % S.nkv, seq = blockIdx.x / S.nkv, key0 = blockIdx.y * BM;
    const int t_begin = cu_seqlens[seq], run = cu_seqlens[seq + 1] - t_begin, start = held[seq], per = S.nh / S.nkv;
    // the run's rows that see some of these keys
    const int row0 = max(0, key0 - start), row1 = S.window > 0 ? min(run, key0 + BM - 1 + S.window - start) : run;
    if (row0 >= row1) return;
    const int nt = (row1 - row0 + BM - 1) / BM, n = per * nt;
    const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
    const uint32_t base = (smem_u32(smem_raw) + 1023u) & ~1023u;
    auto q_smem = [&](int s) { return base + C::TILE + s * C::TILE; };
    const uint32_t bars = smem_u32(s_bars), k_full = bars;
    auto q_full = [&](int s) { return bars + 8u * (1 + s); };
    auto q_empty = [&](int s) { return bars + 8u * (1 + C::STAGES + s); };
    auto s_full = [&](int b) { return bars + 8u * (1 + 2 * C::STAGES + b); };
    auto s_free = [&](int b) { return bars + 8u * (3 + 2 * C::STAGES + b); };
    if (threadIdx.x == 0) {
        s_abort = 0;
        mbar_init(k_full, 1);
        for (int s = 0; s < C::STAGES; ++s) { mbar_init(q_full(s), 1); mbar_init(q_empty(s), 1); }
        for (int b = 0; b < 2; ++b) { mbar_init(s_full(b), 1); mbar_init(s_free(b), 4); }
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 1) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&s_tmem_base)), "r"(2u * BM) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    __syncthreads();
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    tq_grid_launch_dependents();       // behind the allocation: a dependent kernel must not take tensor memory first
    const uint32_t tm = __shfl_sync(0xffffffffu, s_tmem_base, 0);
    auto wait = [&](uint32_t bar, uint32_t parity) { return (bool)__all_sync(0xffffffffu, mbar_wait(bar, parity, &s_abort)); };
    if (warp == 0) {
        const uint32_t elected = elect_one();
        const int pages = min(2, (start + run - 1) / PAGE - key0 / PAGE + 1), first = first_page(start, S.window);
        if (elected) {
            mbar_expect_tx(k_full, (uint32_t)(pages * C::PAGE_BYTES));
            for (int p = 0; p < pages; ++p)
#pragma unroll
                for (int c = 0; c < C::KB; ++c)
                    tma_load_2d(base + c * (BM * 128) + p * (PAGE * 128), &map_k, c * 64, ((seq * S.width + max(key0 / PAGE + p - first, 0)) * 2 * S.nkv + g) * PAGE, k_full);      // (a page no row sees: any other's keys)
        }
        int i = 0;
        for (; i < n; ++i) {
            const int st = i % C::STAGES;
            if (!wait(q_empty(st), ((uint32_t)(i / C::STAGES) & 1u) ^ 1u)) break;
            if (elected) {
                mbar_expect_tx(q_full(st), (uint32_t)C::TILE);
#pragma unroll
                for (int c = 0; c < C::KB; ++c)
                    tma_load_2d(q_smem(st) + c * (BM * 128), &map_q, (g * per + i / nt) * DK + c * 64, t_begin + row0 + i % nt * BM, q_full(st));
            }
        }
        if (s_abort) {                 // let the copies this warp started land before the CTA goes away (bounded)
            for (uint32_t j = 0; j < WAIT_LIMIT && !mbar_try_wait(k_full, 0); ++j) {}
            for (int k = max(0, i - C::STAGES); k < i; ++k)
                for (uint32_t j = 0; j < WAIT_LIMIT && !mbar_try_wait(q_full(k % C::STAGES), (uint32_t)(k / C::STAGES) & 1u); ++j) {}
        }
    } else if (warp == 1) {
        const uint32_t elected = elect_one(), id = idesc(BM, 0);
        const uint64_t kd = desc_k_major(base), qd0 = desc_k_major(q_smem(0));
        bool ok = wait(k_full, 0);
        for (int i = 0; ok && i < n; ++i) {
            const int st = i % C::STAGES, b = i & 1;
            ok = wait(q_full(st), (uint32_t)(i / C::STAGES) & 1u) && (i < 2 || wait(s_free(b), (uint32_t)((i >> 1) - 1) & 1u));
            if (!ok) break;
            asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
            const uint64_t qd = qd0 + (uint64_t)(st * (C::TILE / 16));
#pragma unroll
            for (int k = 0; k < DK / 16; ++k)               // descriptors count in 16 bytes
                umma(tm + (uint32_t)(b * BM), kd + (k / 4) * (BM * 8) + (k % 4) * 2, qd + (k / 4) * (BM * 8) + (k % 4) * 2, id, k > 0 ? 1u : 0u, elected);
            umma_commit(q_empty(st), elected);
            umma_commit(s_full(b), elected);
        }
    } else {
        const int group = (warp - 2) >> 2, quarter = warp & 3, mine = quarter * 32 + lane, key = key0 + mine;
        const uint32_t addr = tm + (uint32_t)(group * BM) + ((uint32_t)(quarter * 32) << 16);
        const tq_f32x2 ff = tq_pack2(S.factor, S.factor);
        tq_f32x2 sum[2] = {tq_pack2(0.f, 0.f), tq_pack2(0.f, 0.f)};
        bool ok = true;
        for (int i = group; ok && i < n; i += 2) {
            const int rb = row0 + i % nt * BM, h = g * per + i / nt, cols = min(BM, row1 - rb), place0 = start + rb;
            __syncwarp();                                       // the previous tile's denominators have been read
#pragma unroll
            for (int c = lane; c < BM; c += 32) s_lse[warp - 2][c] = c < cols ? -lse[(size_t)(t_begin + rb + c) * S.nh + h] : 0.f;
            __syncwarp();
            ok = wait(s_full(group), (uint32_t)(i >> 1) & 1u);
            if (!ok) break;
            asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
            // columns from .. to - 1 see this key
            const int from = key - place0, to = min(cols, S.window > 0 ? key + S.window - place0 : BM);
            const bool whole = cols == BM && key0 + BM - 1 <= place0 && (S.window <= 0 || key0 + S.window >= place0 + BM);
#pragma unroll 1
            for (int c0 = 0; c0 < BM; c0 += 32) {
                uint32_t v[32];
                tmem_ld32(addr + c0, v);
                asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
                const float4* l4 = reinterpret_cast<const float4*>(&s_lse[warp - 2][c0]);
#pragma unroll
                for (int e = 0; e < 32; e += 4) {
                    const float4 l = l4[e / 4];
                    float2 x = tq_unpack2(tq_fma2(tq_pack2(__uint_as_float(v[e]), __uint_as_float(v[e + 1])), ff, tq_pack2(l.x, l.y)));
                    float2 y = tq_unpack2(tq_fma2(tq_pack2(__uint_as_float(v[e + 2]), __uint_as_float(v[e + 3])), ff, tq_pack2(l.z, l.w)));
                    if (!whole) {
                        auto seen = [&](int c) { return c0 + e + c >= from && c0 + e + c < to; };
                        x = make_float2(seen(0) ? x.x : -INFINITY, seen(1) ? x.y : -INFINITY);
                        y = make_float2(seen(2) ? y.x : -INFINITY, seen(3) ? y.y : -INFINITY);
                    }
                    sum[0] = tq_add2(sum[0], tq_pack2(ex2(x.x), ex2(x.y)));
                    sum[1] = tq_add2(sum[1], tq_pack2(ex2(y.x), ex2(y.y)));
                }
            }
            asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
            __syncwarp();
            if (lane == 0) mbar_arrive(s_free(group));
        }
        const float2 a = tq_unpack2(tq_add2(sum[0], sum[1]));
        s_sum[group][mine] = a.x + a.y;
    }
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    __syncthreads();
    if (warp == 1) {
        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(s_tmem_base), "r"(2u * BM) : "memory");
    }
    if (s_abort) {
        if (threadIdx.x == 0) atomicExch(status, 1);
        return;
    }
    if (threadIdx.x < BM) {
        const int key = key0 + (int)threadIdx.x;
        if (key < start + run && !(S.window > 0 && key + S.window <= start)) {
            const int page = TQ_CHECKED(page_table[(size_t)seq * S.table_stride + TQ_CHECKED(key / PAGE, S.table_stride, TQ_IDX_TABLE_COLUMN)], S.n_pages, TQ_IDX_PAGE);
            float* w = weights + ((size_t)page * S.nkv + g) * PAGE + key % PAGE;
            *w = (key < start ? *w : 0.f) + (s_sum[0][threadIdx.x] + s_sum[1][threadIdx.x]);
        }
    }
}

template <int DK>
int launch_weigh_prompt(const CUtensorMap& mq, const CUtensorMap& mk, const WShape& S, const int* cu, const int* held, const int* table, const float* lse, float* weights,
                        int* status, int n_seqs, int tiles, cudaStream_t stream) {
    static std::atomic<unsigned long long> asked{0};
    const cudaError_t e = tq_reserve_smem(weigh8_prompt_kernel<DK>, WCfg<DK>::SMEM_BYTES, asked);
    if (e != cudaSuccess) TQ_FAIL(-1, "weigh8_prompt: cannot reserve %d bytes of shared memory: %s", WCfg<DK>::SMEM_BYTES, cudaGetErrorString(e));
    tq_launch(dim3(S.nkv * n_seqs, tiles), W_THREADS, WCfg<DK>::SMEM_BYTES, stream)(weigh8_prompt_kernel<DK>, mq, mk, S, cu, held, table, lse, weights, status);
    TQ_CHECK_LAUNCH("weigh8_prompt");
    return 0;
}

}  // namespace

// dense [n_seqs * dense_width, 2, nkv, 64, hd] bfloat16: page n of sequence s at s * dense_width + n - the first page its rows see, which
// dense_table [n_seqs, width] says; lost [n_seqs, nkv, width] bytes.  Pages the step does not see are left alone in all three.
TQ_EXPORT int tq_expand8(const void* codes, const void* scales, const int* cu_seqlens, const int* held, const int* page_table, int table_stride, int page_size,
                         int window, void* dense, int* dense_table, void* lost, int width, int dense_width, int n_pages, int n_seqs, int nkv, int hd, cudaStream_t stream) {
    if (n_seqs == 0 || width == 0) return 0;
    int rc = c8_check("expand8", codes, scales, page_size, n_pages, nkv, hd, table_stride);
    if (rc) return rc;
    TQ_REQUIRE(page_size == PAGE && n_seqs <= 65535 && nkv <= 65535 && window >= 0, "expand8: page size %d, %d sequences, %d heads, window %d", page_size, n_seqs, nkv, window);
    TQ_REQUIRE(dense_width >= 1 && dense_width <= width && (long long)n_seqs * width < (1ll << 31) && (uintptr_t)dense % 16 == 0, "expand8: %d pages for each of %d sequences", width, n_seqs);
    const Cache8 c = c8_cache(codes, scales, page_table, table_stride, page_size, n_pages, nkv, hd);
    tq_launch(dim3(width, nkv, n_seqs), 256, 0, stream)(expand8_kernel, c, cu_seqlens, held, window, (uint4*)dense, dense_table, (uint8_t*)lost, width, dense_width);
    TQ_CHECK_LAUNCH("expand8");
    return 0;
}

// q [T, nh, hd] bfloat16, dense as tq_expand8 leaves it, lse [T, nh]: the base-2 logarithm of each row's denominator.  weights [n_pages, nkv, 64]
// of places below held[s] grow by, those of the step's own rows become, the sum over the step's rows and the head's query heads of their weight.
TQ_EXPORT int tq_weigh8_prompt(const void* q, const void* dense, int dense_width, const int* cu_seqlens, const int* held, const int* page_table, int table_stride,
                               int window, float scale, const float* lse, float* weights, int n_pages, int T_, int n_seqs, int max_kv_len, int nh, int nkv, int hd,
                               int* status, cudaStream_t stream) {
    if (n_seqs == 0 || T_ == 0 || max_kv_len == 0) return 0;
    TQ_REQUIRE((hd == 64 || hd == 128) && nkv >= 1 && nh % nkv == 0, "weigh8_prompt: %d heads of %d, %d key/value heads", nh, hd, nkv);
    TQ_REQUIRE(window >= 0 && max_kv_len >= 1 && status != nullptr, "weigh8_prompt: window %d, %d places", window, max_kv_len);
    TQ_REQUIRE(((uintptr_t)q | (uintptr_t)dense) % 16 == 0, "weigh8_prompt: q and the scratch must be 16-byte aligned");
    const int tiles = (max_kv_len + BM - 1) / BM;
    const long long rows = (long long)n_seqs * dense_width * 2 * nkv * PAGE;
    TQ_REQUIRE(rows < (1ll << 31) && tiles <= 65535 && (long long)nkv * n_seqs < (1ll << 31), "weigh8_prompt: %d pages for each of %d sequences", dense_width, n_seqs);
    const WShape S{nh, nkv, dense_width, window, table_stride, n_pages, scale * 1.4426950408889634f};
    CUtensorMap mq, mk;
    int rc = make_map(&mq, q, (uint64_t)T_, (uint64_t)nh * hd, BM, "weigh8_prompt");
    if (!rc) rc = make_map(&mk, dense, (uint64_t)rows, (uint64_t)hd, PAGE, "weigh8_prompt");
    if (rc) return rc;
    return hd == 64 ? launch_weigh_prompt<64>(mq, mk, S, cu_seqlens, held, page_table, lse, weights, status, n_seqs, tiles, stream)
                    : launch_weigh_prompt<128>(mq, mk, S, cu_seqlens, held, page_table, lse, weights, status, n_seqs, tiles, stream);
}
