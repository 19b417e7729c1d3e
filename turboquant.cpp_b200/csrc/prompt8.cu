// Prompts over the 8-bit cache (layout and codes: cache8.cuh).
//
//   tq_expand8   the pages a step sees as bfloat16 pages of a scratch cache, which the tensor-core prompt kernel then reads
#include "cache8.cuh"

TQ_DEFINE_LAST_ERROR

namespace {

constexpr int PAGE = 64;

// ---------------------------------------------------------------------------------------
// A page of one key/value head, both planes.  e4m3 times a power of two is a bfloat16 value: nothing is rounded (below 2^-133 apart).  Rows
// behind the sequence's last become zeros, since the prompt kernel reads whole pages; pages that hold a NaN among the values are marked.
// ---------------------------------------------------------------------------------------
__device__ __forceinline__ uint32_t bf16x2_of(uint32_t two, float scale) {
    const uint32_t h = c8_half2(two);
    float lo, hi;
    asm("{\n\t.reg .b16 l, h;\n\tmov.b32 {l, h}, %2;\n\tcvt.f32.f16 %0, l;\n\tcvt.f32.f16 %1, h;\n\t}" : "=f"(lo), "=f"(hi) : "r"(h));
    const __nv_bfloat162 b = __floats2bfloat162_rn(lo * scale, hi * scale);
    return *reinterpret_cast<const uint32_t*>(&b);
}

__global__ void __launch_bounds__(256) expand8_kernel(Cache8 c, const int* __restrict__ cu_seqlens, const int* __restrict__ held, int window, uint4* __restrict__ dense,
                                                      int* __restrict__ dense_table, uint8_t* __restrict__ lost, int width) {
    tq_grid_wait();                    // everything below may read what the previous kernel wrote
    tq_grid_launch_dependents();
    const int n = blockIdx.x, g = blockIdx.y, seq = blockIdx.z, start = held[seq], run = cu_seqlens[seq + 1] - cu_seqlens[seq], last = start + run - 1;
    if (run <= 0 || n * PAGE > last || n < (window > 0 ? max(0, start + 1 - window) : 0) / PAGE) return;
    const int page = c.page_of(seq, n * PAGE), to = seq * width + n, vecs = c.hd / 16, rows = min(PAGE, last + 1 - n * PAGE);
    bool nan = false;
    for (int i = threadIdx.x; i < 2 * PAGE * vecs; i += 256) {
        const int plane = i / (PAGE * vecs), r = i / vecs % PAGE, v = i % vecs;
        uint4 a = make_uint4(0, 0, 0, 0), b = a;
        if (r < rows) {
            const uint4 x = *reinterpret_cast<const uint4*>(c.codes + c.codes_at(page, plane, g) + (size_t)r * c.hd + v * 16);
            const float s = c8_scale(c.scales[c.scales_at(page, plane, g) + r / C8_BLOCK]);
            a = make_uint4(bf16x2_of(x.x & 0xffffu, s), bf16x2_of(x.x >> 16, s), bf16x2_of(x.y & 0xffffu, s), bf16x2_of(x.y >> 16, s));
            b = make_uint4(bf16x2_of(x.z & 0xffffu, s), bf16x2_of(x.z >> 16, s), bf16x2_of(x.w & 0xffffu, s), bf16x2_of(x.w >> 16, s));
            const uint32_t u[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
            for (int k = 0; k < 4; ++k) nan |= plane == 1 && (((u[k] & 0x7f7f7f7fu) + 0x01010101u) & 0x80808080u) != 0;
        }
        uint4* d = dense + (((size_t)to * 2 + plane) * c.nkv + g) * (PAGE * vecs * 2) + (size_t)r * vecs * 2 + v * 2;
        d[0] = a;
        d[1] = b;
    }
    const bool any = __syncthreads_or(nan);
    if (threadIdx.x == 0) {
        lost[((size_t)seq * c.nkv + g) * width + n] = any ? 1 : 0;
        if (g == 0) dense_table[to] = to;
    }
}

}  // namespace

// dense [n_seqs * width, 2, nkv, 64, hd] bfloat16: page n of sequence s at s * width + n, which dense_table [n_seqs, width] says;
// lost [n_seqs, nkv, width] bytes.  Pages the step does not see are left alone in all three.
TQ_EXPORT int tq_expand8(const void* codes, const void* scales, const int* cu_seqlens, const int* held, const int* page_table, int table_stride, int page_size,
                         int window, void* dense, int* dense_table, void* lost, int width, int n_pages, int n_seqs, int nkv, int hd, cudaStream_t stream) {
    if (n_seqs == 0 || width == 0) return 0;
    int rc = c8_check("expand8", codes, scales, page_size, n_pages, nkv, hd, table_stride);
    if (rc) return rc;
    TQ_REQUIRE(page_size == PAGE && n_seqs <= 65535 && nkv <= 65535 && window >= 0, "expand8: page size %d, %d sequences, %d heads, window %d", page_size, n_seqs, nkv, window);
    TQ_REQUIRE((long long)n_seqs * width < (1ll << 31) && (uintptr_t)dense % 16 == 0, "expand8: %d pages for each of %d sequences", width, n_seqs);
    const Cache8 c{(uint8_t*)codes, (uint8_t*)scales, page_table, table_stride, page_size, n_pages, nkv, hd};
    tq_launch(dim3(width, nkv, n_seqs), 256, 0, stream)(expand8_kernel, c, cu_seqlens, held, window, (uint4*)dense, dense_table, (uint8_t*)lost, width);
    TQ_CHECK_LAUNCH("expand8");
    return 0;
}
