// tb_paged.cuh — what the paged cache's kernels share (include/tb_gguf_dequant.h
// part 4): the device view of one layer's pages and of a step's ragged batch, and
// element conversion.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "tb_common.cuh"
#include "tb_internal.h"

namespace tb {

// One layer of the cache, strides in elements.
struct KvView {
    const void *k, *v;
    long long page_stride, head_stride, pos_stride;
    int n_pages, page_size, n_kv_heads;
    FastDiv page_div;   // position / page_size
};

struct KvBatch {
    const int *start, *len, *pages;
    int n_seqs, n_tokens, pages_stride, pages_width;
};

struct KvRows {
    const void *p;
    long long row, head;
};

// Launchers (tb_paged.cu, tb_kvattn.cu): arguments checked by the C entry
// points; 1 = launched (attention: the number of launches).  hd: head_dim, ti / tc: types of the rows and the cache.
int rope_table_launch(float *t, int n_pos, int rot, double base, double factor, double fast, double slow,
                      double orig_len, double attn, int mode, cudaStream_t st);
int kv_append_launch(const KvView &c, const KvBatch &b, int hd, int ti, int tc, int nh, const KvRows &q,
                     const KvRows &k, const KvRows &v, const KvRows &o, const float *table, const float *qn,
                     const float *kn, int n_pos, int rot, int inter, float eps, int *err, int sms, cudaStream_t st);
int kv_copy_launch(void *k, void *v, int esize, int n_layers, int n_pages, int page_size, int n_kv_heads, int hd,
                   long long layer_stride, long long page_stride, long long head_stride, long long pos_stride,
                   const int *src, const int *dst, int n, cudaStream_t st);
size_t kv_attend_ws();
int kv_attend_launch(const KvView &c, const KvBatch &b, int hd, int ti, int tc, int nh, const KvRows &q,
                     const KvRows &o, float scale, int window, int sinks, int max_new, int max_len, void *ws, int *err,
                     int sms, uint32_t wait_limit, cudaStream_t st);

// Launch with programmatic stream serialization: the kernels of the paged cache
// begin with griddepcontrol.wait (after what needs no other kernel's data), so a
// launch's start-up overlaps the end of the one before it.  Nothing that a kernel may
// write is read by __ldg: the grid lives while the one before it still writes, and such a
// load may be moved ahead of the wait.  1 = launched.
inline int kv_launch(const void *fn, dim3 grid, unsigned threads, size_t smem, void **args, cudaStream_t st)
{
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = grid;
    cfg.blockDim = dim3(threads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = st;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    if (cudaLaunchKernelExC(&cfg, fn, args) == cudaSuccess) return 1;
    cudaGetLastError();
    return 0;
}

// Element types as template arguments.
template <int T> struct KvType;
template <> struct KvType<QT_F32> { using E = float; };
template <> struct KvType<QT_F16> { using E = __half; };
template <> struct KvType<QT_BF16> { using E = __nv_bfloat16; };

__device__ __forceinline__ float kv_f(float x) { return x; }
__device__ __forceinline__ float kv_f(__half x) { return __half2float(x); }
__device__ __forceinline__ float kv_f(__nv_bfloat16 x) { return __bfloat162float(x); }

// 8 consecutive elements (16-byte aligned) as fp32, and back with one rounding.
__device__ __forceinline__ void kv_load8(const float *p, float (&x)[8])
{
    const float4 a = *reinterpret_cast<const float4 *>(p), b = *reinterpret_cast<const float4 *>(p + 4);
    x[0] = a.x, x[1] = a.y, x[2] = a.z, x[3] = a.w, x[4] = b.x, x[5] = b.y, x[6] = b.z, x[7] = b.w;
}
__device__ __forceinline__ void kv_load8(const __half *p, float (&x)[8])
{
    const uint4 a = *reinterpret_cast<const uint4 *>(p);
    const uint32_t w[4] = {a.x, a.y, a.z, a.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float2 f = __half22float2(*reinterpret_cast<const __half2 *>(&w[i]));
        x[2 * i] = f.x, x[2 * i + 1] = f.y;
    }
}
__device__ __forceinline__ void kv_load8(const __nv_bfloat16 *p, float (&x)[8])
{
    const uint4 a = *reinterpret_cast<const uint4 *>(p);
    const uint32_t w[4] = {a.x, a.y, a.z, a.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        x[2 * i] = __uint_as_float(w[i] << 16);
        x[2 * i + 1] = __uint_as_float(w[i] & 0xFFFF0000u);
    }
}
__device__ __forceinline__ void kv_store8(float *p, const float (&x)[8])
{
    *reinterpret_cast<float4 *>(p) = make_float4(x[0], x[1], x[2], x[3]);
    *reinterpret_cast<float4 *>(p + 4) = make_float4(x[4], x[5], x[6], x[7]);
}
__device__ __forceinline__ void kv_store8(__half *p, const float (&x)[8])
{
    __half2 h[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) h[i] = __floats2half2_rn(x[2 * i], x[2 * i + 1]);
    *reinterpret_cast<uint4 *>(p) = *reinterpret_cast<const uint4 *>(h);
}
__device__ __forceinline__ void kv_store8(__nv_bfloat16 *p, const float (&x)[8])
{
    __nv_bfloat162 h[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) h[i] = __floats2bfloat162_rn(x[2 * i], x[2 * i + 1]);
    *reinterpret_cast<uint4 *>(p) = *reinterpret_cast<const uint4 *>(h);
}

__device__ __forceinline__ void kv_store1(float *p, float x) { *p = x; }
__device__ __forceinline__ void kv_store1(__half *p, float x) { *p = __float2half_rn(x); }
__device__ __forceinline__ void kv_store1(__nv_bfloat16 *p, float x) { *p = __float2bfloat16_rn(x); }

// Sequence s of the batch: its new rows [row0, row0 + n) and its length.
// False (and the error word set) when they cannot be.
struct KvSeq {
    int row0, n, len;
};
__device__ __forceinline__ bool kv_seq(const KvBatch &b, const KvView &c, int s, KvSeq &q, int *err)
{
    const int a = b.start[s], e = b.start[s + 1];
    q.row0 = a;
    q.n = e - a;
    q.len = b.len[s];
    // (lengths near 2^31 would overflow where they are rounded up to tiles)
    const bool ok = a >= 0 && e >= a && e <= b.n_tokens && q.len >= 0 && q.len <= 0x7FFFFF00 && q.n <= q.len &&
                    q.len <= static_cast<long long>(b.pages_width) * c.page_size;
    if (!ok && err) atomicExch(err, ERR_RUNTIME);
    return ok;
}

// Element offset of position p of sequence s for kv head h; -1 (and the error
// word set) when its page lies outside the pool.
__device__ __forceinline__ long long kv_at(const KvBatch &b, const KvView &c, int s, int p, int h, int *err)
{
    const uint32_t pi = fdiv(static_cast<uint32_t>(p), c.page_div);
    const int page = b.pages[static_cast<long long>(s) * b.pages_stride + pi];
    if (page < 0 || page >= c.n_pages) {
        if (err) atomicExch(err, ERR_RUNTIME);
        return -1;
    }
    return page * c.page_stride + h * c.head_stride + (p - static_cast<int>(pi) * c.page_size) * c.pos_stride;
}

// Which positions a row at position i sees: [0, first) and [lo, i + 1).
struct KvSpan {
    int first, lo;
};
__host__ __device__ __forceinline__ KvSpan kv_span(int i, int window, int sinks)
{
    KvSpan s{0, 0};
    if (window > 0 && i - window + 1 > 0) {
        s.lo = i - window + 1;
        s.first = sinks < s.lo ? sinks : s.lo;
    }
    return s;
}

}  // namespace tb
