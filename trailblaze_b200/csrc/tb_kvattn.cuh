// tb_kvattn.cuh — what the two attention kernels over the paged cache share.
#pragma once

#include <cmath>
#include <cstdio>
#include <type_traits>

#include "tb_paged.cuh"
#include "tb_tc.cuh"

namespace tb {

struct AttnArgs {
    KvView c;
    KvBatch b;
    KvRows q, o;
    int nh, group, window, sinks;
    float scale2;   // scale * log2(e)
    int *err;
    uint32_t wait_limit;
    int ax_pos, ax_head, ax_page;   // the tensor maps' axes 1..3: which of them is which
    float *part;                    // [gridDim.x] partial results
    unsigned *arrived;              // [gridDim.x] arrival counters, zero between calls
    int many_rows;                  // k_kv_few: sequences of more rows are the other launch's
};

// The launch of k_kv_many (tb_kvmany.cu) for the sequences of more than few_rows
// query rows per kv head; 1 = launched, -1 = q's strides rule it out.
static constexpr int kManyCtas = 160;
size_t kv_many_part_bytes();   // a partial result
int kv_many_launch(AttnArgs a, int hd, int tc, int few_rows, int sms, cudaStream_t st);

__device__ __forceinline__ float ex2(float x)   // 2^x, 2 ulp; 0 for -inf
{
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ void prefetch_map(const CUtensorMap *m)
{
    asm volatile("prefetch.tensormap [%0];" ::"l"(reinterpret_cast<uint64_t>(m)) : "memory");
}

__device__ __forceinline__ void tma_load_4d(uint32_t dst, const CUtensorMap *map, int x, int y, int z, int w, uint32_t bar)
{
    asm volatile("cp.async.bulk.tensor.4d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, "
                 "%5}], [%6];" ::"r"(dst),
                 "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(y), "r"(z), "r"(w), "r"(bar)
                 : "memory");
}

// Division of counts that are 64 bits wide by type and 32 by size: a 64-bit division
// takes some hundred instructions, which a launch of a few microseconds sees.
__device__ __forceinline__ unsigned long long kv_div(unsigned long long a, unsigned long long b)
{
    if (((a | b) >> 32) == 0) return static_cast<uint32_t>(a) / static_cast<uint32_t>(b);
    return a / b;
}

// total units of work in G parts that differ by one at most, the longer ones first.
struct KvShare {
    unsigned long long base;
    unsigned rem;
    __device__ __forceinline__ KvShare(unsigned long long total, unsigned G) : base(kv_div(total, G)), rem(static_cast<unsigned>(total - base * G)) {}
    __device__ __forceinline__ unsigned long long start(unsigned c) const { return base * c + min(c, rem); }
    __device__ __forceinline__ unsigned of(unsigned long long unit) const   // the part that holds a unit
    {
        const unsigned long long longer = (base + 1) * rem;
        return static_cast<unsigned>(unit < longer ? kv_div(unit, base + 1) : rem + kv_div(unit - longer, base));
    }
};

// The rows of sequences whose numbers contradict each other: the error word, and
// zeros as far as the rows exist (one CTA, all its threads).
template <int HD, class I>
__device__ void kv_zero_bad(const AttnArgs &a)
{
    for (int s = 0; s < a.b.n_seqs; ++s) {
        KvSeq q;
        if (kv_seq(a.b, a.c, s, q, a.err)) continue;
        const int lo = max(0, a.b.start[s]), hi = min(a.b.n_tokens, a.b.start[s + 1]);
        const long long n = static_cast<long long>(max(0, hi - lo)) * a.nh * HD;
        for (long long e = threadIdx.x; e < n; e += blockDim.x) {
            const long long th = e / HD;
            kv_store1(static_cast<I *>(const_cast<void *>(a.o.p)) + (lo + th / a.nh) * a.o.row + (th % a.nh) * a.o.head +
                          e % HD,
                      0.f);
        }
    }
}

// The layer's K and V as 4-D tensors: dimension, then position in the page, head
// and page in order of their strides (ax: which axis each became).  Boxes of
// 128 bytes by box_rows positions, 128-byte swizzle; pages outside the pool read
// as zeros.
inline bool kv_maps(const KvView &c, int hd, int tc, int box_rows, CUtensorMap *k, CUtensorMap *v, int (&ax)[3])
{
    EncodeTiled enc = encode_tiled();
    if (!enc) {
        fprintf(stderr, "[tb_cuda] kv_attend: cuTensorMapEncodeTiled not available\n");
        return false;
    }
    const cuuint64_t es = tc == QT_F32 ? 4 : 2;
    cuuint64_t size[3] = {static_cast<cuuint64_t>(c.page_size), static_cast<cuuint64_t>(c.n_kv_heads),
                          static_cast<cuuint64_t>(c.n_pages)};
    cuuint64_t stride[3] = {static_cast<cuuint64_t>(c.pos_stride) * es, static_cast<cuuint64_t>(c.head_stride) * es,
                            static_cast<cuuint64_t>(c.page_stride) * es};
    int order[3] = {0, 1, 2};
    for (int i = 0; i < 3; ++i)
        for (int j = i + 1; j < 3; ++j)
            if (stride[order[j]] < stride[order[i]]) {
                const int x = order[i];
                order[i] = order[j];
                order[j] = x;
            }
    cuuint64_t dims[4] = {static_cast<cuuint64_t>(hd)}, strides[3];
    cuuint32_t box[4] = {static_cast<cuuint32_t>(128 / es), 1, 1, 1};
    const cuuint32_t estr[4] = {1, 1, 1, 1};
    for (int i = 0; i < 3; ++i) {
        ax[order[i]] = i;
        dims[i + 1] = size[order[i]];
        strides[i] = stride[order[i]];
        if (order[i] == 0) box[i + 1] = static_cast<cuuint32_t>(box_rows);
    }
    const CUtensorMapDataType type = tc == QT_F32   ? CU_TENSOR_MAP_DATA_TYPE_FLOAT32
                                     : tc == QT_F16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16
                                                    : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16;
    for (int i = 0; i < 2; ++i) {
        const CUresult r = enc(i ? v : k, type, 4, const_cast<void *>(i ? c.v : c.k), dims, strides, box, estr,
                               CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                               CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
        if (r != CUDA_SUCCESS) {
            fprintf(stderr, "[tb_cuda] kv_attend: tensor map encode failed (%d)\n", static_cast<int>(r));
            return false;
        }
    }
    return true;
}

}  // namespace tb
