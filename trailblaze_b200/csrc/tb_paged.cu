// tb_paged.cu — operators of the paged cache other than attention: rotary
// append and page copies, and the rotary table (include/tb_gguf_dequant.h
// part 4).
#include <cstdio>
#include <vector>

#include "tb_paged.cuh"

namespace tb {

// ---- the rotary table ----
struct RopeArgs {
    float *t;
    int n_pos, half, mode;
    double base, factor, fast, slow, orig_len, attn;
    int rot;
};

// One thread per (position, pair), everything in 64 bits and rounded once: an
// fp32 angle of 10^5 radians would be off by 4e-3.
__global__ void __launch_bounds__(256) k_rope_table(const RopeArgs a)
{
    const long long n = static_cast<long long>(a.n_pos) * a.half;
    for (long long e = blockIdx.x * 256ll + threadIdx.x; e < n; e += gridDim.x * 256ll) {
        const int i = static_cast<int>(e % a.half);
        const double pos = static_cast<double>(e / a.half);
        const double base = a.mode == 2 ? a.base * pow(a.factor, a.rot / (a.rot - 2.0)) : a.base;
        double f = pow(base, -2.0 * i / a.rot);
        if (a.mode == 1) f /= a.factor;
        if (a.mode == 3) {
            const double turns = a.orig_len * f / 6.283185307179586476925;
            const double g = fmin(fmax((turns - a.slow) / (a.fast - a.slow), 0.0), 1.0);
            f *= g + (1.0 - g) / a.factor;
        }
        double s, c;
        sincos(pos * f, &s, &c);
        reinterpret_cast<float2 *>(a.t)[e] =
            make_float2(static_cast<float>(c * a.attn), static_cast<float>(s * a.attn));
    }
}

int rope_table_launch(float *t, int n_pos, int rot, double base, double factor, double fast, double slow,
                      double orig_len, double attn, int mode, cudaStream_t st)
{
    const NvtxRange nvtx("tb.rope_table");
    const long long n = static_cast<long long>(n_pos) * (rot / 2);
    const long long blocks = (n + 255) / 256;
    k_rope_table<<<static_cast<unsigned>(blocks < 148 * 64 ? blocks : 148 * 64), 256, 0, st>>>(
        RopeArgs{t, n_pos, rot / 2, mode, base, factor, fast, slow, orig_len, attn, rot});
    return cudaGetLastError() == cudaSuccess ? 1 : 0;
}

// ---- append ----
struct AppendArgs {
    KvView c;
    KvBatch b;
    KvRows q, k, v, o;
    const float *table, *qn, *kn;
    int n_pos, rot, inter, nh;
    float eps;
    int *err;
};

// CTA (token, part of the heads): 8 elements a lane, so HD / 8 lanes hold a head
// and a warp 32 * 8 / HD heads.  A lane's dimensions are the same for every head
// that it visits, so the token's cos and sin sit in its registers:
//   y[d] = x[d] cos + x[partner] sin', sin' negative for a pair's first element.
// Interleaved pairs lie in one lane; halves are exchanged through shared memory,
// which takes any rot_dim.
template <int HD, int TI, int TC>
__global__ void __launch_bounds__(256) k_kv_append(const AppendArgs a)
{
    using I = typename KvType<TI>::E;
    using C = typename KvType<TC>::E;
    constexpr int L = HD / 8, HW = 32 / L;   // lanes a head, heads a warp
    __shared__ int s_at;
    __shared__ __align__(16) float xs[8 * HW][HD];
    const int t = blockIdx.x, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int s = kv_seq_of_row(a.b, t, &s_at, a.err);
    if (s < 0) return;   // a row of no sequence
    KvSeq q;
    const bool ok = kv_seq(a.b, a.c, s, q, a.err);
    const int pos = q.len - q.n + (t - q.row0);
    long long at = -1;
    if (ok && (!a.table || pos < a.n_pos)) at = kv_at(a.b, a.c, s, pos, 0, a.err);
    else if (ok && threadIdx.x == 0) atomicExch(a.err, ERR_RUNTIME);
    const int grp = lane / L, d0 = (lane % L) * 8;   // the lane's head of the warp's, its first dimension
    float cs[8], sn[8];
    int partner[8];
    const int half = a.rot / 2;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        const int d = d0 + e;
        cs[e] = 1.f, sn[e] = 0.f, partner[e] = -1;
        if (a.table && at >= 0 && d < a.rot) {
            const bool second = a.inter ? (d & 1) : d >= half;
            const int pair = a.inter ? d >> 1 : second ? d - half : d;
            partner[e] = a.inter ? d ^ 1 : second ? d - half : d + half;
            const float2 w = __ldg(reinterpret_cast<const float2 *>(a.table) + static_cast<long long>(pos) * half + pair);
            cs[e] = w.x;
            sn[e] = second ? w.y : -w.y;
        }
    }
    const int items = a.nh + a.c.n_kv_heads;
    for (int base = (blockIdx.y * 8 + warp) * HW; base < items; base += gridDim.y * 8 * HW) {
        const int it = base + grp;
        const bool on = it < items, isq = it < a.nh;
        const int h = isq ? it : it - a.nh;
        const KvRows &src = isq ? a.q : a.k;
        float x[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) x[e] = 0.f;
        if (on) kv_load8(static_cast<const I *>(src.p) + t * src.row + h * src.head + d0, x);
        const float *nw = isq ? a.qn : a.kn;
        float ss = 0.f;
#pragma unroll
        for (int e = 0; e < 8; ++e) ss = fmaf(x[e], x[e], ss);
#pragma unroll
        for (int o = L / 2; o > 0; o >>= 1) ss += __shfl_xor_sync(0xFFFFFFFFu, ss, o);
        if (nw) {
            const float sc = 1.0f / sqrtf(ss / static_cast<float>(HD) + a.eps);
            float w[8];
            kv_load8(nw + d0, w);
#pragma unroll
            for (int e = 0; e < 8; ++e) x[e] = x[e] * sc * w[e];
        }
        float *mine = xs[warp * HW + grp];
        kv_store8(mine + d0, x);
        __syncwarp();
        float y[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) y[e] = partner[e] >= 0 ? fmaf(mine[partner[e]], sn[e], x[e] * cs[e]) : x[e];
        __syncwarp();
        if (!on) continue;
        if (isq) {
            if (at < 0) {
#pragma unroll
                for (int e = 0; e < 8; ++e) y[e] = 0.f;
            }
            kv_store8(static_cast<I *>(const_cast<void *>(a.o.p)) + t * a.o.row + h * a.o.head + d0, y);
        } else if (at >= 0) {
            const long long to = at + h * a.c.head_stride + d0;
            kv_store8(static_cast<C *>(const_cast<void *>(a.c.k)) + to, y);
            kv_load8(static_cast<const I *>(a.v.p) + t * a.v.row + h * a.v.head + d0, x);
            kv_store8(static_cast<C *>(const_cast<void *>(a.c.v)) + to, x);
        }
    }
}

template <int HD, int TI>
static void *append_kernel(int tc)
{
    return tc == QT_F32 ? reinterpret_cast<void *>(k_kv_append<HD, TI, QT_F32>)
         : tc == QT_F16 ? reinterpret_cast<void *>(k_kv_append<HD, TI, QT_F16>)
                        : reinterpret_cast<void *>(k_kv_append<HD, TI, QT_BF16>);
}

int kv_append_launch(const KvView &c, const KvBatch &b, int hd, int ti, int tc, int nh, const KvRows &q,
                     const KvRows &k, const KvRows &v, const KvRows &o, const float *table, const float *qn,
                     const float *kn, int n_pos, int rot, int inter, float eps, int *err, int sms, cudaStream_t st)
{
    const NvtxRange nvtx("tb.kv_append");
    if (b.n_tokens == 0) return 1;
    AppendArgs a{c, b, q, k, v, o, table, qn, kn, n_pos, rot, inter, nh, eps, err};
    void *fn = hd == 128 ? (ti == QT_F32 ? append_kernel<128, QT_F32>(tc) : ti == QT_F16 ? append_kernel<128, QT_F16>(tc)
                                                                                  : append_kernel<128, QT_BF16>(tc))
                         : (ti == QT_F32 ? append_kernel<64, QT_F32>(tc) : ti == QT_F16 ? append_kernel<64, QT_F16>(tc)
                                                                                 : append_kernel<64, QT_BF16>(tc));
    // few tokens: their heads over several CTAs, one pass of the warps each
    const int passes = (nh + c.n_kv_heads + 8 * (256 / hd) - 1) / (8 * (256 / hd));
    int parts = 4 * sms / b.n_tokens;
    parts = parts < 1 ? 1 : parts > passes ? passes : parts;
    void *args[] = {&a};
    if (cudaLaunchKernel(fn, dim3(b.n_tokens, parts), dim3(256), args, 0, st) != cudaSuccess) {
        cudaGetLastError();
        return 0;
    }
    return 1;
}

// ---- page copies ----
static constexpr int kCopyPairs = 480;   // per launch: the pairs travel as a kernel argument

struct CopyArgs {
    char *k, *v;
    long long layer_stride, page_stride;    // bytes
    long long run, cnt0, str0, cnt1, str1;  // a page: cnt1 x cnt0 runs of run bytes
    int n_layers, n;
    int src[kCopyPairs], dst[kCopyPairs];
};

// CTA (pair, K or V, layer): one page of one tensor.
__global__ void __launch_bounds__(256) k_kv_copy(const __grid_constant__ CopyArgs a)
{
    const int i = blockIdx.x;
    char *base = (blockIdx.y ? a.v : a.k) + blockIdx.z * a.layer_stride;
    const char *from = base + a.src[i] * a.page_stride;
    char *to = base + a.dst[i] * a.page_stride;
    const long long rv = a.run / 16, total = rv * a.cnt0 * a.cnt1;
    for (long long u = threadIdx.x; u < total; u += 256) {
        const long long w = u % rv, r = u / rv;
        const long long off = w * 16 + (r % a.cnt0) * a.str0 + (r / a.cnt0) * a.str1;
        *reinterpret_cast<uint4 *>(to + off) = *reinterpret_cast<const uint4 *>(from + off);
    }
}

int kv_copy_launch(void *k, void *v, int esize, int n_layers, int n_pages, int page_size, int n_kv_heads, int hd,
                   long long layer_stride, long long page_stride, long long head_stride, long long pos_stride,
                   const int *src, const int *dst, int n, cudaStream_t st)
{
    const NvtxRange nvtx("tb.kv_copy");
    try {
        // a destination is given once and is no source
        std::vector<unsigned char> seen(static_cast<size_t>(n_pages), 0);
        for (int i = 0; i < n; ++i) {
            if (src[i] < 0 || src[i] >= n_pages || dst[i] < 0 || dst[i] >= n_pages) return 0;
            seen[src[i]] |= 1;
        }
        for (int i = 0; i < n; ++i) {
            if (seen[dst[i]]) return 0;
            seen[dst[i]] = 2;
        }
    } catch (const std::exception &e) {
        fprintf(stderr, "[tb_cuda] kv_copy: %s\n", e.what());
        return 0;
    }
    CopyArgs a{};
    a.k = static_cast<char *>(k);
    a.v = static_cast<char *>(v);
    a.layer_stride = layer_stride * esize;
    a.page_stride = page_stride * esize;
    a.n_layers = n_layers;
    // a page as runs: the head's row, then the inner and the outer of heads and positions
    long long run = static_cast<long long>(hd) * esize;
    long long c0 = page_size, s0 = pos_stride * esize, c1 = n_kv_heads, s1 = head_stride * esize;
    if (s1 < s0) {
        const long long tc = c0, ts = s0;
        c0 = c1, s0 = s1, c1 = tc, s1 = ts;
    }
    if (s0 == run) {   // contiguous: one longer run
        run *= c0;
        c0 = c1, s0 = s1, c1 = 1, s1 = 0;
        if (s0 == run) run *= c0, c0 = 1, s0 = 0;
    }
    a.run = run, a.cnt0 = c0, a.str0 = s0, a.cnt1 = c1, a.str1 = s1;
    for (int i0 = 0; i0 < n; i0 += kCopyPairs) {
        a.n = n - i0 < kCopyPairs ? n - i0 : kCopyPairs;
        for (int i = 0; i < a.n; ++i) a.src[i] = src[i0 + i], a.dst[i] = dst[i0 + i];
        k_kv_copy<<<dim3(a.n, 2, n_layers), 256, 0, st>>>(a);
        if (cudaGetLastError() != cudaSuccess) return 0;
    }
    return 1;
}

}  // namespace tb
