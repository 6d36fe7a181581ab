// tb_kvattn.cu — attention of a step's new tokens over the paged cache
// (include/tb_gguf_dequant.h part 4, tb_cuda_kv_attend_dev).
#include <cmath>
#include <cstdio>

#include "tb_paged.cuh"

namespace tb {

struct AttnArgs {
    KvView c;
    KvBatch b;
    KvRows q, o;
    int nh, window, sinks;
    float scale2;   // scale * log2(e)
    int *err;
};

// One warp per (row, head), fp32, a position at a time.
template <int HD, int TI, int TC>
__global__ void __launch_bounds__(256) k_kv_rows(const AttnArgs a)
{
    using I = typename KvType<TI>::E;
    using C = typename KvType<TC>::E;
    constexpr int D = HD / 32;
    __shared__ int s_at;
    const int t = blockIdx.x, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int s = kv_seq_of_row(a.b, t, &s_at, a.err);
    if (s < 0) return;
    KvSeq sq;
    const bool ok = kv_seq(a.b, a.c, s, sq, a.err);
    const int pos = sq.len - sq.n + (t - sq.row0);
    for (int h = blockIdx.y * 8 + warp; h < a.nh; h += gridDim.y * 8) {
        float q[D], acc[D], m, l;
        const I *qp = static_cast<const I *>(a.q.p) + t * a.q.row + h * a.q.head + lane * D;
#pragma unroll
        for (int d = 0; d < D; ++d) q[d] = kv_f(qp[d]) * a.scale2;
        kv_row_attend<HD, C>(a.b, a.c, s, h / (a.nh / a.c.n_kv_heads), pos, 0, ok ? sq.len : 0, a.window, a.sinks, q, m,
                             l, acc, a.err);
        I *op = static_cast<I *>(const_cast<void *>(a.o.p)) + t * a.o.row + h * a.o.head + lane * D;
#pragma unroll
        for (int d = 0; d < D; ++d) kv_store1(op + d, m == -INFINITY ? 0.f : acc[d] / l);
    }
}

template <int HD, int TI>
static void *rows_kernel(int tc)
{
    return tc == QT_F32 ? reinterpret_cast<void *>(k_kv_rows<HD, TI, QT_F32>)
         : tc == QT_F16 ? reinterpret_cast<void *>(k_kv_rows<HD, TI, QT_F16>)
                        : reinterpret_cast<void *>(k_kv_rows<HD, TI, QT_BF16>);
}

size_t kv_attend_ws() { return 16; }

int kv_attend_launch(const KvView &c, const KvBatch &b, int hd, int ti, int tc, int nh, const KvRows &q,
                     const KvRows &o, float scale, int window, int sinks, int max_new, int max_len, void *ws, int *err,
                     int sms, cudaStream_t st)
{
    const NvtxRange nvtx("tb.kv_attend");
    (void)max_new, (void)max_len, (void)ws, (void)sms;
    if (b.n_tokens == 0) return 1;
    AttnArgs a{c, b, q, o, nh, window, sinks, scale * 1.4426950408889634f, err};
    void *fn = hd == 128 ? (ti == QT_F32 ? rows_kernel<128, QT_F32>(tc) : ti == QT_F16 ? rows_kernel<128, QT_F16>(tc)
                                                                                : rows_kernel<128, QT_BF16>(tc))
                         : (ti == QT_F32 ? rows_kernel<64, QT_F32>(tc) : ti == QT_F16 ? rows_kernel<64, QT_F16>(tc)
                                                                               : rows_kernel<64, QT_BF16>(tc));
    void *args[] = {&a};
    if (cudaLaunchKernel(fn, dim3(b.n_tokens, (nh + 7) / 8), dim3(256), args, 0, st) != cudaSuccess) {
        cudaGetLastError();
        return 0;
    }
    return 1;
}

}  // namespace tb
