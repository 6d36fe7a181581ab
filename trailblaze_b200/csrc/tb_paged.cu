// tb_paged.cu — operators of the paged cache other than attention: rotary
// append and page copies, and the rotary table (include/tb_gguf_dequant.h
// part 4).
#include <cstdio>
#include <type_traits>
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
    int parts;   // warps a token
};

// One warp per token, or per part of a token's heads when tokens are few; 8
// elements a lane, so HD / 8 lanes hold a head and a warp HW = 256 / HD of them.  A
// lane's dimensions are the same for every head that it visits, so the token's cos
// and sin (and the norm's weights) sit in its registers:
//   y[d] = x[d] cos + x[partner] sin', sin' negative for a pair's first element;
// a dimension that does not rotate has cos = 1 and a partner of zero.  Interleaved
// pairs lie in one lane; a half's partners are loaded a second time (they are in L1 by
// then; shuffles took twice the instructions).  The rows' bytes bound it, and next the
// instructions, hence the forms of the loop: norm or not; no rotation, pairs, halves
// whose partners lie 8 together, or halves that split a lane's 8.  8192 tokens of 32 q
// and 8 kv bf16 heads, half of each rotated: 47 us, 4.3 TB/s of 6.5 that a copy
// reaches; one token: 4.3 us, the launch and a chain of five loads.
enum AppendMode { TURN_NONE, TURN_PAIRS, TURN_HALVES, TURN_SPLIT };

template <class E>
struct Raw {   // 8 elements
    uint4 v[sizeof(E) / 2];
    __device__ __forceinline__ void load(const E *p)
    {
#pragma unroll
        for (int i = 0; i < static_cast<int>(sizeof(E) / 2); ++i) v[i] = reinterpret_cast<const uint4 *>(p)[i];
    }
    __device__ __forceinline__ void clear()
    {
#pragma unroll
        for (int i = 0; i < static_cast<int>(sizeof(E) / 2); ++i) v[i] = make_uint4(0, 0, 0, 0);
    }
    __device__ __forceinline__ void set(int e, E x) { reinterpret_cast<E *>(v)[e] = x; }
    __device__ __forceinline__ void to(float (&x)[8]) const { kv_load8(reinterpret_cast<const E *>(v), x); }
};

template <int HD, int TI, int TC>
__global__ void __launch_bounds__(256, 2) k_kv_append(const __grid_constant__ AppendArgs a)
{
    using I = typename KvType<TI>::E;
    using C = typename KvType<TC>::E;
    constexpr int L = HD / 8, HW = 32 / L, U = 4;   // lanes a head, heads a warp, heads ahead
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    asm volatile("griddepcontrol.wait;" ::: "memory");
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    if (blockIdx.x == 0)   // ranges that cannot be are reported once, whatever tokens they claim
        for (int s = threadIdx.x; s < a.b.n_seqs; s += 256) {
            KvSeq q;
            kv_seq(a.b, a.c, s, q, a.err);
        }
    const uint32_t w = blockIdx.x * 8u + warp, wt = w / static_cast<uint32_t>(a.parts);
    if (wt >= static_cast<uint32_t>(a.b.n_tokens)) return;
    const int t = static_cast<int>(wt), part = static_cast<int>(w - wt * a.parts);
    const int d0 = (lane % L) * 8, grp = lane / L, step = a.parts * HW;
    // passes of HW heads, q's, then k's, then v's: this warp's are part, part + parts, ...
    const int nk = a.c.n_kv_heads, pq = (a.nh + HW - 1) / HW, pk = (nk + HW - 1) / HW;
    auto first = [&](int p) { return (part >= p ? part : part + (p - part + a.parts - 1) / a.parts * a.parts) - p; };
    const int h0 = part * HW + grp, hk = first(pq) * HW + grp, hv = first(pq + pk) * HW + grp;
    const int half = a.rot / 2, n_turn = a.table ? min(8, max(0, a.rot - d0)) : 0;   // of the lane's 8, those that rotate
    const int mode = !a.table ? TURN_NONE : a.inter ? TURN_PAIRS : (half & 7) == 0 ? TURN_HALVES : TURN_SPLIT;
    const int mate = n_turn == 0 ? 0 : d0 >= half ? -half : half;   // TURN_HALVES
    Raw<I> x[U], z[U];
#pragma unroll
    for (int u = 0; u < U; ++u) z[u].clear();
    auto load = [&](auto mode_, const I *p, long long inc, int h, int n) {
        constexpr int MODE = decltype(mode_)::value;
#pragma unroll
        for (int u = 0; u < U; ++u)
            if (h + u * step < n) {
                x[u].load(p + u * inc);
                if constexpr (MODE == TURN_HALVES)
                    if (n_turn > 0) z[u].load(p + u * inc + mate);
                if constexpr (MODE == TURN_SPLIT) {
#pragma unroll
                    for (int e = 0; e < 8; ++e)
                        if (e < n_turn) z[u].set(e, p[u * inc + e + (d0 + e >= half ? -half : half)]);
                }
            }
        __syncwarp();   // q_out may be q: nothing is stored before its partner is read
    };
    const I *qp = static_cast<const I *>(a.q.p) + t * a.q.row + h0 * a.q.head + d0;
    if (h0 < a.nh) asm volatile("prefetch.global.L1 [%0];" ::"l"(qp));   // on its way during the look-up
    // ---- the token's sequence, position, page and angles ----
    int s;
    if (a.b.n_seqs <= 32) {
        const unsigned hit = __ballot_sync(0xFFFFFFFFu, lane < a.b.n_seqs && a.b.start[lane] <= t && t < a.b.start[lane + 1]);
        s = __ffs(hit) - 1;
    } else {   // the first sequence that ends after t
        int lo = 0, hi = a.b.n_seqs;
        while (lo < hi) {
            const int mid = (lo + hi) >> 1;
            if (a.b.start[mid + 1] > t) hi = mid;
            else lo = mid + 1;
        }
        s = lo < a.b.n_seqs && a.b.start[lo] <= t ? lo : -1;
    }
    if (s < 0) return;   // a row of no sequence
    KvSeq sq;
    const bool ok = kv_seq(a.b, a.c, s, sq, a.err);
    const int pos = sq.len - sq.n + (t - sq.row0);
    long long at = -1;
    if (ok && (!a.table || pos < a.n_pos)) at = kv_at(a.b, a.c, s, pos, 0, a.err);
    else if (ok && lane == 0) atomicExch(a.err, ERR_RUNTIME);
    if (at < 0) {   // nowhere to go: zeros for q
        const float zero[8] = {};
        I *op = static_cast<I *>(const_cast<void *>(a.o.p)) + t * a.o.row + d0;
        for (int h = h0; h < a.nh; h += step) kv_store8(op + h * a.o.head, zero);
        return;
    }
    float cs[8], sn[8];
    const float2 *angles = reinterpret_cast<const float2 *>(a.table) + static_cast<long long>(pos) * half;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        const int d = d0 + e;
        cs[e] = 1.f, sn[e] = 0.f;
        if (e < n_turn) {
            const bool second = a.inter ? (e & 1) : d >= half;
            const float2 v = angles[a.inter ? d >> 1 : second ? d - half : d];
            cs[e] = v.x;
            sn[e] = second ? v.y : -v.y;
        }
    }
    float wd[8], wm[8];   // a norm's weights at this lane's dimensions and at their partners
    // heads h, h + step, ... of n, from p to o
    auto heads = [&](auto norm_, auto mode_, const I *p, long long inc, auto *o, long long o_inc, int h, int n, const float *nw) {
        constexpr bool NORM = decltype(norm_)::value;
        constexpr int MODE = decltype(mode_)::value;
        if constexpr (NORM) {   // this norm's weights, in the place of the last one's
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const int d = d0 + e, m = e >= n_turn ? d : MODE == TURN_PAIRS ? d ^ 1 : d >= half ? d - half : d + half;
                wd[e] = nw[d];
                wm[e] = nw[m];
            }
        }
        for (; h - grp < n; h += U * step, p += U * inc, o += U * o_inc) {
            load(mode_, p, inc, h, n);
#pragma unroll
            for (int u = 0; u < U; ++u) {
                float y[8], w[8];
                x[u].to(y);
                float sc = 1.f;
                if constexpr (NORM) {
                    float ss = 0.f;
#pragma unroll
                    for (int e = 0; e < 8; ++e) ss = fmaf(y[e], y[e], ss);
#pragma unroll
                    for (int k = L / 2; k > 0; k >>= 1) ss += __shfl_xor_sync(0xFFFFFFFFu, ss, k);
                    sc = 1.0f / sqrtf(ss / static_cast<float>(HD) + a.eps);
                }
                if constexpr (NORM) {
#pragma unroll
                    for (int e = 0; e < 8; ++e) y[e] *= sc * wd[e];
                }
                if constexpr (MODE == TURN_PAIRS) {
#pragma unroll
                    for (int e = 0; e < 8; ++e) w[e] = e < n_turn ? y[e ^ 1] : 0.f;
                } else if constexpr (MODE != TURN_NONE) {
                    z[u].to(w);
                    if constexpr (NORM) {
#pragma unroll
                        for (int e = 0; e < 8; ++e) w[e] *= sc * wm[e];
                    }
                }
#pragma unroll
                for (int e = 0; e < 8; e += 2) {
                    if constexpr (MODE == TURN_NONE) break;
                    const float2 r = __ffma2_rn(make_float2(w[e], w[e + 1]), make_float2(sn[e], sn[e + 1]),
                                                __fmul2_rn(make_float2(y[e], y[e + 1]), make_float2(cs[e], cs[e + 1])));
                    y[e] = r.x, y[e + 1] = r.y;
                }
                if (h + u * step < n) kv_store8(o + u * o_inc, y);
            }
        }
    };
    I *op = static_cast<I *>(const_cast<void *>(a.o.p)) + t * a.o.row + h0 * a.o.head + d0;
    const I *kp = static_cast<const I *>(a.k.p) + t * a.k.row + hk * a.k.head + d0;
    const I *vp = static_cast<const I *>(a.v.p) + t * a.v.row + hv * a.v.head + d0;
    C *kc = static_cast<C *>(const_cast<void *>(a.c.k)) + at + hk * a.c.head_stride + d0;
    C *vc = static_cast<C *>(const_cast<void *>(a.c.v)) + at + hv * a.c.head_stride + d0;
    const long long q_inc = step * a.q.head, k_inc = step * a.k.head, v_inc = step * a.v.head;
    const long long o_inc = step * a.o.head, c_inc = step * a.c.head_stride;
    using std::integral_constant;
    auto all = [&](auto MODE) {
        using T1 = integral_constant<bool, true>;
        using T0 = integral_constant<bool, false>;
        if (a.qn) heads(T1(), MODE, qp, q_inc, op, o_inc, h0, a.nh, a.qn);
        else heads(T0(), MODE, qp, q_inc, op, o_inc, h0, a.nh, a.qn);
        if (a.kn) heads(T1(), MODE, kp, k_inc, kc, c_inc, hk, nk, a.kn);
        else heads(T0(), MODE, kp, k_inc, kc, c_inc, hk, nk, a.kn);
        heads(T0(), integral_constant<int, TURN_NONE>(), vp, v_inc, vc, c_inc, hv, nk, nullptr);
    };
    if (mode == TURN_HALVES) all(integral_constant<int, TURN_HALVES>());
    else if (mode == TURN_PAIRS) all(integral_constant<int, TURN_PAIRS>());
    else if (mode == TURN_NONE) all(integral_constant<int, TURN_NONE>());
    else all(integral_constant<int, TURN_SPLIT>());
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
    // A token's heads over several warps until the GPU has two waves of 16 an SM, at most
    // a pass each (8192 tokens of 48 heads: 47 us with four heads ahead at two CTAs an SM,
    // 52 with two at three CTAs and four waves, 105 with a CTA a token).
    const int hw = 256 / hd, passes = (nh + hw - 1) / hw + 2 * ((c.n_kv_heads + hw - 1) / hw);
    const int parts = (2 * 16 * sms + b.n_tokens - 1) / b.n_tokens;
    a.parts = parts > passes ? passes : parts;
    const long long warps = static_cast<long long>(b.n_tokens) * a.parts;
    void *args[] = {&a};
    return kv_launch(fn, dim3(static_cast<unsigned>((warps + 7) / 8)), 256, 0, args, st);
}

// ---- page copies ----
static constexpr int kCopyPairs = 480;   // per launch: the pairs travel as a kernel argument

struct CopyArgs {
    char *k, *v;
    long long layer_stride, page_stride;    // bytes
    long long str0, str1;                   // a page: runs of run * 16 bytes, cnt0 of them str0 apart, these str1 apart
    uint32_t vecs, piece;                   // 16-byte pieces of a page; how many of them a CTA copies
    FastDiv run, cnt0;
    int src[kCopyPairs], dst[kCopyPairs];
};

// CTA (pair and part of the page, K or V, layer).  Bound by the bytes, read and
// written once: 384 pages of 64 KB in 36 layers, K and V (3.6 GB both ways) in 562 us,
// 6.45 TB/s; 3 pages in 4.7 us, of which 2.9 are bytes.
template <bool WHOLE>   // a page is one run
__global__ void __launch_bounds__(256) k_kv_copy(const __grid_constant__ CopyArgs a)
{
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    asm volatile("griddepcontrol.wait;" ::: "memory");
    const uint32_t parts = (a.vecs + a.piece - 1) / a.piece, i = blockIdx.x / parts, part = blockIdx.x - i * parts;
    char *base = (blockIdx.y ? a.v : a.k) + blockIdx.z * a.layer_stride;
    const char *from = base + a.src[i] * a.page_stride;
    char *to = base + a.dst[i] * a.page_stride;
    const uint32_t end = min(a.vecs, (part + 1) * a.piece);
    auto at = [&](uint32_t u) -> long long {
        if (WHOLE) return u * 16ll;
        const uint32_t r = fdiv(u, a.run), r1 = fdiv(r, a.cnt0);
        return (u - r * a.run.d) * 16ll + (r - r1 * a.cnt0.d) * a.str0 + r1 * a.str1;
    };
    uint32_t u = part * a.piece + threadIdx.x;
    for (; u + 3 * 256 < end; u += 4 * 256) {
        uint4 x[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) x[k] = __ldcs(reinterpret_cast<const uint4 *>(from + at(u + k * 256)));
#pragma unroll
        for (int k = 0; k < 4; ++k) *reinterpret_cast<uint4 *>(to + at(u + k * 256)) = x[k];
    }
    for (; u < end; u += 256) *reinterpret_cast<uint4 *>(to + at(u)) = __ldcs(reinterpret_cast<const uint4 *>(from + at(u)));
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
    const long long vecs = run / 16 * c0 * c1;
    if (vecs > 0x40000000) return 0;   // a page of 16 GB
    const bool whole = c0 == 1 && c1 == 1;
    a.vecs = static_cast<uint32_t>(vecs);
    a.run = make_fastdiv(static_cast<uint32_t>(run / 16));
    a.cnt0 = make_fastdiv(static_cast<uint32_t>(c0));
    a.str0 = s0, a.str1 = s1;
    // 16 KB a CTA while that leaves the GPU room, else 64 KB: a fork's few pages spread
    // over all SMs, and many pages do not pay for a CTA's start every 16 KB
    const long long small = static_cast<long long>(n) * 2 * n_layers * ((vecs + 1023) / 1024);
    a.piece = small <= 16 * 148 ? 1024 : 4096;
    const uint32_t parts = (a.vecs + a.piece - 1) / a.piece;
    const int per = static_cast<int>(0x7FFFFFFF / parts) < kCopyPairs ? static_cast<int>(0x7FFFFFFF / parts) : kCopyPairs;
    for (int i0 = 0; i0 < n; i0 += per) {
        const int m = n - i0 < per ? n - i0 : per;
        for (int i = 0; i < m; ++i) a.src[i] = src[i0 + i], a.dst[i] = dst[i0 + i];
        void *args[] = {&a};
        if (!kv_launch(whole ? reinterpret_cast<void *>(k_kv_copy<true>) : reinterpret_cast<void *>(k_kv_copy<false>),
                       dim3(m * parts, 2, n_layers), 256, 0, args, st))
            return 0;
    }
    return 1;
}

}  // namespace tb
