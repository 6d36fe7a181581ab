// tb_kvattn.cuh — what the attention kernels over the paged cache share.
#pragma once

#include <cmath>
#include <cstdio>
#include <type_traits>

#include "tb_paged.cuh"
#include "tb_tc.cuh"

namespace tb {

// Bound of the waits after a failed one, for what is still in flight (copies into
// shared memory, MMAs): it is no part of the wait limit, which a user may set, since a
// CTA that ended before its copies landed would leave them to the next one's memory.
static constexpr uint32_t kKvDrain = 1u << 26;

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
    int *arrived;                   // [gridDim.x] arrival counters, zero between calls: see kv_await
    int many_rows;                  // k_kv_few: sequences of more rows are the other launch's
};

// The launch of k_kv_many (tb_kvmany.cu) for the sequences of more than few_rows
// query rows per kv head; 1 = launched, -1 = q's strides rule it out.
static constexpr int kManyCtas = 160;
size_t kv_many_part_bytes();   // a partial result
int kv_many_launch(AttnArgs a, int hd, int tc, int few_rows, int sms, cudaStream_t st);
// The same of k_kv_tf32 (tb_kvtf32.cu), for any types.
size_t kv_tf32_part_bytes();
int kv_tf32_launch(AttnArgs a, int hd, int ti, int tc, int few_rows, int sms, cudaStream_t st);

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

// ---- mma.sync and its operands ----
// None of these is volatile, so that the compiler can load ahead of the products.
// What keeps the loads inside a stage's use: their addresses derive from a
// shared_after() behind the wait for the stage, and pin() of the results stands
// before the stage is given back.
__device__ __forceinline__ void pin(float (&x)[4])
{
    asm volatile("" : "+f"(x[0]), "+f"(x[1]), "+f"(x[2]), "+f"(x[3])::"memory");
}
__device__ __forceinline__ void ldsm4(uint32_t a, uint32_t (&r)[4])
{
    asm("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(a));
}
__device__ __forceinline__ void ldsm4t(uint32_t a, uint32_t (&r)[4])
{
    asm("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(a));
}
__device__ __forceinline__ uint32_t mat_t(uint32_t x)   // transpose of an 8 x 8 matrix of 16-bit elements
{
    uint32_t y;
    asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
    return y;
}
template <int TC>
__device__ __forceinline__ void mma16(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1)
{
    if constexpr (TC == QT_BF16)
        asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
                     "{%0, %1, %2, %3};"
                     : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                     : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
    else
        asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
                     "{%0, %1, %2, %3};"
                     : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                     : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void mma_tf32(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1)
{
    asm("mma.sync.aligned.m16n8k8.row.col.f32.tf32.tf32.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
                 "{%0, %1, %2, %3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
// x = hi + lo, hi rounded to tf32 (10 bits of mantissa); the tensor core reads
// lo's upper 19 bits: what is lost lies 2^-21 below x and has no preferred sign.
__device__ __forceinline__ void split_tf32(uint32_t x, uint32_t &hi, uint32_t &lo)
{
    hi = (x + 0x1000u) & 0xFFFFE000u;
    lo = __float_as_uint(__uint_as_float(x) - __uint_as_float(hi));
}
// Two fp32 as a pair of 16-bit elements, and what the rounding left over.
template <int TC>
__device__ __forceinline__ uint32_t pack16(float &x, float &y)
{
    uint32_t w;
    if constexpr (TC == QT_BF16) {
        const __nv_bfloat162 h = __floats2bfloat162_rn(x, y);
        w = *reinterpret_cast<const uint32_t *>(&h);
        x -= __uint_as_float(w << 16);
        y -= __uint_as_float(w & 0xFFFF0000u);
    } else {
        const __half2 h = __floats2half2_rn(x, y);
        w = *reinterpret_cast<const uint32_t *>(&h);
        const float2 f = __half22float2(h);
        x -= f.x;
        y -= f.y;
    }
    return w;
}

// ---- TMEM ----
#define TB_R32(r)                                                                                                       \
    "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),       \
        "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(r[16]), "r"(r[17]), "r"(r[18]),     \
        "r"(r[19]), "r"(r[20]), "r"(r[21]), "r"(r[22]), "r"(r[23]), "r"(r[24]), "r"(r[25]), "r"(r[26]), "r"(r[27]),     \
        "r"(r[28]), "r"(r[29]), "r"(r[30]), "r"(r[31])
#define TB_W32(c, r)                                                                                                    \
    c(r[0]), c(r[1]), c(r[2]), c(r[3]), c(r[4]), c(r[5]), c(r[6]), c(r[7]), c(r[8]), c(r[9]), c(r[10]), c(r[11]),       \
        c(r[12]), c(r[13]), c(r[14]), c(r[15]), c(r[16]), c(r[17]), c(r[18]), c(r[19]), c(r[20]), c(r[21]), c(r[22]),   \
        c(r[23]), c(r[24]), c(r[25]), c(r[26]), c(r[27]), c(r[28]), c(r[29]), c(r[30]), c(r[31])
#define TB_LIST32                                                                                                       \
    "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, %17, %18, %19, %20, %21, %22, %23, "   \
    "%24, %25, %26, %27, %28, %29, %30, %31}"
__device__ __forceinline__ void tmem_ld32(uint32_t at, uint32_t *r)
{
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x32.b32 " TB_LIST32 ", [%32];" : TB_W32("=r", r) : "r"(at) : "memory");
}
__device__ __forceinline__ void tmem_st32(uint32_t at, const uint32_t *r)
{
    asm volatile("tcgen05.st.sync.aligned.32x32b.x32.b32 [%32], " TB_LIST32 ";" ::TB_R32(r), "r"(at) : "memory");
}
// The loads before it are complete; the registers pass through, so that nothing
// that uses them moves ahead.
__device__ __forceinline__ void tmem_wait_ld(uint32_t *r)
{
    asm volatile("tcgen05.wait::ld.sync.aligned;" : TB_W32("+r", r)::"memory");
}
__device__ __forceinline__ void after_wait(uint32_t *r) { asm volatile("" : TB_W32("+r", r)::"memory"); }
__device__ __forceinline__ void tmem_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

// R rows of one kv head again, in fp32, over their visible positions in [j0, j1) only, by the
// whole warp: for rows whose result is not finite, where a NaN or an infinity may have come
// from a position that the row does not see.  q: the rows; i: their positions (-1: none).
// m: the largest exponent of 2 (-inf: nothing seen), l: the sum of the numerators, acc: the
// weighted sums of dimensions lane % (HD / 8) * 8 ....
// An infinity in V at the start of a long prompt sends every row here, so: 32 positions at a
// time, HD / 8 lanes a position (a load takes whole rows), U loads in flight, R rows to a
// load.  Where a numerator is NaN so is all of its row; once all rows are, the rest need not
// be looked at.
template <int HD, class I, class E, int R, int U>
__device__ __forceinline__ void kv_rows_attend(const AttnArgs &a, const I *const (&q)[R], int s, int h, const int (&i)[R], int j0,
                                               int j1, float (&m)[R], float (&l)[R], float (&acc)[R][8])
{
    constexpr int LR = HD / 8, RW = 32 / LR;   // lanes a row, rows a load
    const int lane = threadIdx.x & 31, d0 = lane % LR * 8, grp = lane / LR;
    const E *kp = static_cast<const E *>(a.c.k) + d0, *vp = static_cast<const E *>(a.c.v) + d0;
    float qq[R][8];
    KvSpan sp[R];
    int first = 0, lo = 0x7FFFFFFF, last = -1;   // of all rows
    unsigned open = 0;                           // rows that are not NaN yet
#pragma unroll
    for (int r = 0; r < R; ++r) {
        sp[r] = kv_span(max(i[r], 0), a.window, a.sinks);
        if (i[r] >= 0) first = max(first, sp[r].first), lo = min(lo, sp[r].lo), open |= 1u << r;
        last = max(last, i[r]);
        kv_load8(q[r] + d0, qq[r]);
#pragma unroll
        for (int d = 0; d < 8; ++d) qq[r][d] *= a.scale2;   // before the products: they may leave fp32 without
        m[r] = -INFINITY, l[r] = 0.f;
#pragma unroll
        for (int d = 0; d < 8; ++d) acc[r][d] = 0.f;
    }
    j1 = min(j1, last + 1);
    for (int j = j0; j < j1 && open; j += 32) {
        if (j >= first && j < lo) j = min(lo, j1);   // the stretch that is hidden from all
        const int p = j + lane;
        const long long at = p < j1 && (p < first || p >= lo) ? kv_at(a.b, a.c, s, p, h, a.err) : -1;
        float x[R], w[R];
        unsigned see[R];
#pragma unroll
        for (int r = 0; r < R; ++r) {
            const bool on = at >= 0 && p <= i[r] && (p < sp[r].first || p >= sp[r].lo);
            x[r] = -INFINITY;
            see[r] = __ballot_sync(0xFFFFFFFFu, on);
        }
#pragma unroll 1
        for (int k0 = 0; k0 < 32; k0 += U * RW) {
            float kk[U][8];
#pragma unroll
            for (int u = 0; u < U; ++u) {   // (a position that is none: any row that there is)
                const long long ka = __shfl_sync(0xFFFFFFFFu, at, k0 + u * RW + grp);
                kv_load8(kp + (ka < 0 ? 0 : ka), kk[u]);
            }
#pragma unroll
            for (int r = 0; r < R; ++r) {
                float sc[U];
#pragma unroll
                for (int u = 0; u < U; ++u) {
                    float2 t = make_float2(0.f, 0.f);
#pragma unroll
                    for (int d = 0; d < 8; d += 2)
                        t = __ffma2_rn(make_float2(qq[r][d], qq[r][d + 1]), make_float2(kk[u][d], kk[u][d + 1]), t);
                    sc[u] = t.x + t.y;
                }
                // the U sums over a row's lanes together: at each step a lane keeps half of them, so
                // that lane u * (LR / U) of a row's has the u-th in the end
                int o = LR / 2;
#pragma unroll
                for (int n = U / 2; n > 0; n >>= 1, o >>= 1)
#pragma unroll
                    for (int u = 0; u < n; ++u) {
                        const bool up = lane & o;
                        const float keep = up ? sc[u + n] : sc[u], send = up ? sc[u] : sc[u + n];
                        sc[u] = keep + __shfl_xor_sync(0xFFFFFFFFu, send, o);
                    }
                for (; o > 0; o >>= 1) sc[0] += __shfl_xor_sync(0xFFFFFFFFu, sc[0], o);
                const float mine = __shfl_sync(0xFFFFFFFFu, sc[0], lane % RW * LR + lane / RW % U * (LR / U));
                if (lane / (U * RW) == k0 / (U * RW) && (see[r] >> lane & 1u)) x[r] = mine;
            }
        }
#pragma unroll
        for (int r = 0; r < R; ++r) {
            float top = x[r];   // fmaxf passes NaN over
#pragma unroll
            for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xFFFFFFFFu, top, o));
            top = fmaxf(top, m[r]);
            const float corr = m[r] == -INFINITY ? 0.f : exp2f(m[r] - top);
            w[r] = x[r] == -INFINITY ? 0.f : exp2f(x[r] - top);
            m[r] = top;
            l[r] = l[r] * corr + w[r];
#pragma unroll
            for (int d = 0; d < 8; ++d) acc[r][d] *= corr;
            if (__any_sync(0xFFFFFFFFu, isnan(w[r]))) open &= ~(1u << r);
        }
#pragma unroll 1
        for (int k0 = 0; k0 < 32; k0 += U * RW) {
            float v[U][8];
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const long long va = __shfl_sync(0xFFFFFFFFu, at, k0 + u * RW + grp);
                kv_load8(vp + (va < 0 ? 0 : va), v[u]);
            }
#pragma unroll
            for (int u = 0; u < U; ++u)
#pragma unroll
                for (int r = 0; r < R; ++r) {
                    const int k = k0 + u * RW + grp;
                    const float wk = __shfl_sync(0xFFFFFFFFu, w[r], k);
                    if (see[r] >> k & 1u) {
#pragma unroll
                        for (int d = 0; d < 8; d += 2) {
                            const float2 t = __ffma2_rn(make_float2(wk, wk), make_float2(v[u][d], v[u][d + 1]),
                                                        make_float2(acc[r][d], acc[r][d + 1]));
                            acc[r][d] = t.x, acc[r][d + 1] = t.y;
                        }
                    }
                }
        }
    }
#pragma unroll
    for (int r = 0; r < R; ++r) {
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) l[r] += __shfl_xor_sync(0xFFFFFFFFu, l[r], o);
#pragma unroll
        for (int d = 0; d < 8; ++d) {
#pragma unroll
            for (int o = LR; o < 32; o <<= 1) acc[r][d] += __shfl_xor_sync(0xFFFFFFFFu, acc[r][d], o);
            if (i[r] >= 0 && !(open >> r & 1u)) acc[r][d] = NAN;
        }
    }
}
// Whole rows and their output, those of the lanes of todo (row, head and position: the lane's).
template <int HD, class I, class E>
__device__ __forceinline__ void kv_rows_again(const AttnArgs &a, unsigned todo, int row, int head, int pos, int s, int h)
{
    constexpr int R = 3, U = 4;   // (4 rows are done in 0.8 of the time, and cost the kernel's usual loop 1.5 % by its registers)
    while (todo) {
        const I *qp[R];
        long long to[R];
        int i[R];
#pragma unroll
        for (int r = 0; r < R; ++r) {
            const int src = todo ? __ffs(todo) - 1 : 0;
            const long long t = __shfl_sync(0xFFFFFFFFu, row, src), n = __shfl_sync(0xFFFFFFFFu, head, src);
            i[r] = __shfl_sync(0xFFFFFFFFu, pos, src);
            if (!todo) i[r] = -1;
            qp[r] = static_cast<const I *>(a.q.p) + (todo ? t * a.q.row + n * a.q.head : 0);
            to[r] = t * a.o.row + n * a.o.head;
            todo &= todo - 1;   // (0 stays 0)
        }
        float m[R], l[R], x[R][8];
        kv_rows_attend<HD, I, E, R, U>(a, qp, s, h, i, 0, 0x7FFFFFFF, m, l, x);
#pragma unroll
        for (int r = 0; r < R; ++r) {
#pragma unroll
            for (int d = 0; d < 8; ++d) x[r][d] = l[r] == 0.f ? 0.f : x[r][d] / l[r];
            if (i[r] >= 0 && (threadIdx.x & 31) < HD / 8)
                kv_store8(static_cast<I *>(const_cast<void *>(a.o.p)) + to[r] + (threadIdx.x & 31) * 8, x[r]);
        }
    }
}

// ---- joining the parts of an item ----
// Each part's warps add one to the counter of the CTA that has the item's beginning,
// which waits for all of them and takes that number off again.  Every CTA does its share
// of both, once, after a failed wait as well: a call leaves the counters at zero however
// it ends, since a part that comes after its joiner has given up finds the number gone
// already.
__device__ __forceinline__ void kv_arrive(const AttnArgs &a, int cta)   // by a whole warp, for its stores
{
    __syncwarp();
    if ((threadIdx.x & 31) == 0) {
        __threadfence();
        atomicAdd(a.arrived + cta, 1);
    }
    __syncwarp();
}
// One thread: true when want warps have arrived, false when the limit ran out or stop().
template <class F>
__device__ __forceinline__ bool kv_await(const AttnArgs &a, int cta, int want, F stop)
{
    int n = 0;
    uint32_t i = 0;
    do {
        asm volatile("ld.acquire.gpu.global.s32 %0, [%1];" : "=r"(n) : "l"(a.arrived + cta) : "memory");
    } while (n < want && ++i < a.wait_limit && !stop());
    atomicSub(a.arrived + cta, want);
    return n >= want;
}

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

// ---- row tiles by position tiles: how the chunk kernels cut their work ----
// An item is (sequence, kv head, tpi of its new tokens); its units are tiles of TILE
// positions.  All units end to end, in the order sequence, head, row tile, position,
// are cut into equal parts, one a CTA.
struct KvItem {
    int s, h, rt;           // sequence, kv head, row tile
    KvSeq q;
    int n_rt;               // row tiles a head
    int t0, t1;             // new tokens [t0, t1) of the sequence
    int ns, lo, n;          // its position tiles: [0, ns) and [lo, lo + n - ns)
};

template <int TILE>
__device__ __forceinline__ int kv_item_tiles(const AttnArgs &a, int tpi, const KvSeq &q, int rt, KvItem *it)
{
    const int t0 = rt * tpi, t1 = min(q.n, t0 + tpi), p0 = q.len - q.n;
    const KvSpan sp = kv_span(p0 + t0, a.window, a.sinks);
    const int hi = (p0 + t1 - 1) / TILE + 1;
    int ns = 0, lo = 0, n = hi;
    if (a.sinks < sp.lo) {
        ns = (a.sinks + TILE - 1) / TILE;
        lo = max(sp.lo / TILE, ns);
        n = ns + hi - lo;
    }
    if (it) it->t0 = t0, it->t1 = t1, it->ns = ns, it->lo = lo, it->n = n;
    return n;
}
template <int TILE>
__device__ __forceinline__ int kv_item_pos(const KvItem &it, int j)
{
    return (j < it.ns ? j : j - it.ns + it.lo) * TILE;
}
// True when a row of the item sees any of the positions [p, p + n).  The page of others is not
// looked at: it may have been given away since the window left it.
__device__ __forceinline__ bool kv_item_sees(const AttnArgs &a, const KvItem &it, int p, int n)
{
    return p < it.q.len && (p < a.sinks || p + n > kv_span(it.q.len - it.q.n + it.t0, a.window, a.sinks).lo);
}
// True for a sequence of this launch: one of more rows than few_rows.
__device__ __forceinline__ bool kv_item_seq(const AttnArgs &a, int few_rows, int s, KvSeq &q)
{
    return kv_seq(a.b, a.c, s, q, nullptr) && static_cast<long long>(q.n) * a.group > few_rows && q.n > 0;
}
__device__ __forceinline__ void kv_item_enter(const AttnArgs &a, int tpi, int few_rows, KvItem &it)   // at sequence it.s, or a later one
{
    while (it.s < a.b.n_seqs && !kv_item_seq(a, few_rows, it.s, it.q)) ++it.s;
    it.n_rt = (it.q.n + tpi - 1) / tpi;
}
template <int TILE>
__device__ __forceinline__ void kv_item_next(const AttnArgs &a, int tpi, int few_rows, KvItem &it)
{
    if (++it.rt == it.n_rt) {
        it.rt = 0;
        if (++it.h == a.c.n_kv_heads) {
            it.h = 0;
            ++it.s;
            kv_item_enter(a, tpi, few_rows, it);
        }
    }
    kv_item_tiles<TILE>(a, tpi, it.q, it.rt, &it);
}
// Units of one head of the lane's sequence q (n = 0: none); the whole warp calls it.
// Long chunks' row tiles are counted by all lanes together.
template <int TILE>
__device__ __forceinline__ unsigned long long kv_head_units(const AttnArgs &a, int tpi, const KvSeq &q)
{
    const int lane = threadIdx.x & 31, n_rt = (q.n + tpi - 1) / tpi;
    unsigned long long f = 0;
    if (n_rt <= 4)
        for (int rt = 0; rt < n_rt; ++rt) f += kv_item_tiles<TILE>(a, tpi, q, rt, nullptr);
    for (unsigned todo = __ballot_sync(0xFFFFFFFFu, n_rt > 4); todo; todo &= todo - 1) {
        const int src = __ffs(todo) - 1;
        KvSeq x = q;
        x.n = __shfl_sync(0xFFFFFFFFu, q.n, src);
        x.len = __shfl_sync(0xFFFFFFFFu, q.len, src);
        const int m = __shfl_sync(0xFFFFFFFFu, n_rt, src);
        unsigned long long c = 0;
        for (int rt = lane; rt < m; rt += 32) c += kv_item_tiles<TILE>(a, tpi, x, rt, nullptr);
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) c += __shfl_xor_sync(0xFFFFFFFFu, c, o);
        if (lane == src) f = c;
    }
    return f;
}

struct KvScan {   // shared
    unsigned long long warp[16], items[16], total;
    unsigned parts;           // the CTAs with a share of the total
    int seq, head, rt, off;   // the CTA's first item and its first unit there
};
struct KvCtaShare {
    KvShare share;
    unsigned cta;             // of the units, against blockIdx: a part's CTA starts before the one that waits for it
    unsigned long long u0, u1;
    __device__ __forceinline__ KvCtaShare() : share(1, 1), cta(0), u0(0), u1(0) {}
};

// The CTA's share of all units, by a scan over the sequences; false when it has none.
// The first item is in sh after the caller's next __syncthreads().
// A CTA for every item, or more, with at least MIN units each: what a finer cut saves
// in products it spends on joining parts.
template <int TILE, int MIN, int WARPS, int HD, class I>
__device__ __forceinline__ bool kv_items_share(const AttnArgs &a, int tpi, int few_rows, KvScan &sh, KvCtaShare &my)
{
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int per = (a.b.n_seqs + WARPS * 32 - 1) / (WARPS * 32);
    const int sq0 = min(a.b.n_seqs, tid * per), sq1 = min(a.b.n_seqs, sq0 + per);
    unsigned long long mine = 0, items = 0;
    bool bad_seq = false;
    for (int k = 0; k < per; ++k) {
        KvSeq q{};
        if (sq0 + k < sq1) {
            bad_seq = bad_seq || !kv_seq(a.b, a.c, sq0 + k, q, nullptr);
            if (!kv_item_seq(a, few_rows, sq0 + k, q)) q.n = 0;
        }
        mine += kv_head_units<TILE>(a, tpi, q) * a.c.n_kv_heads;
        items += static_cast<unsigned long long>((q.n + tpi - 1) / tpi) * a.c.n_kv_heads;
    }
    unsigned long long incl = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const unsigned long long x = __shfl_up_sync(0xFFFFFFFFu, incl, o);
        if (lane >= o) incl += x;
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) items += __shfl_xor_sync(0xFFFFFFFFu, items, o);
    if (lane == 31) sh.warp[warp] = incl, sh.items[warp] = items;
    if (__syncthreads_or(bad_seq) && blockIdx.x == 0) kv_zero_bad<HD, I>(a);
    unsigned long long before = incl - mine, total = 0, most = 0;
    for (int w = 0; w < WARPS; ++w) {
        before += w < warp ? sh.warp[w] : 0;
        total += sh.warp[w];
        most += sh.items[w];
    }
    most = max(most, (total + MIN - 1) / MIN);
    const unsigned G = most < gridDim.x ? static_cast<unsigned>(most) : gridDim.x;
    if (blockIdx.x >= G) return false;
    if (tid == 0) sh.total = total, sh.parts = G;
    my.cta = G - 1 - blockIdx.x;
    my.share = KvShare(total, G);
    my.u0 = my.share.start(my.cta), my.u1 = my.share.start(my.cta + 1);
    const unsigned long long u0 = my.u0;
    const bool mine_u0 = before <= u0 && u0 < before + mine;
    if (__any_sync(0xFFFFFFFFu, mine_u0)) {   // the warp whose sequences hold u0
        unsigned long long at = before;
        bool found = false;
        KvSeq fq{};
        int fs = 0;
        unsigned long long fr = 0, ff = 1;
        for (int k = 0; k < per; ++k) {
            KvSeq q{};
            if (sq0 + k < sq1 && !kv_item_seq(a, few_rows, sq0 + k, q)) q.n = 0;
            const unsigned long long f = kv_head_units<TILE>(a, tpi, q), n = f * a.c.n_kv_heads;
            if (mine_u0 && !found && u0 < at + n) found = true, fq = q, fs = sq0 + k, fr = u0 - at, ff = f;
            at += n;
        }
        const int src = __ffs(__ballot_sync(0xFFFFFFFFu, found)) - 1;
        fq.n = __shfl_sync(0xFFFFFFFFu, fq.n, src);
        fq.len = __shfl_sync(0xFFFFFFFFu, fq.len, src);
        const unsigned long long r = __shfl_sync(0xFFFFFFFFu, fr, src), f = __shfl_sync(0xFFFFFFFFu, ff, src);
        const unsigned long long head = kv_div(r, f);
        unsigned long long rem = r - head * f;   // units of the head before u0: the row tile, 32 at a time
        const int n_rt = (fq.n + tpi - 1) / tpi;
        for (int base = 0; base < n_rt; base += 32) {
            const unsigned long long k = base + lane < n_rt ? kv_item_tiles<TILE>(a, tpi, fq, base + lane, nullptr) : 0;
            unsigned long long c = k;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const unsigned long long x = __shfl_up_sync(0xFFFFFFFFu, c, o);
                if (lane >= o) c += x;
            }
            const unsigned hit = __ballot_sync(0xFFFFFFFFu, rem < c);
            if (hit) {
                if (lane == __ffs(hit) - 1) {
                    sh.head = static_cast<int>(head);
                    sh.rt = base + lane;
                    sh.off = static_cast<int>(rem - (c - k));
                }
                break;
            }
            rem -= __shfl_sync(0xFFFFFFFFu, c, 31);
        }
        if (lane == src) sh.seq = fs;
    }
    return true;
}
template <int TILE>
__device__ __forceinline__ KvItem kv_item_first(const AttnArgs &a, int tpi, int few_rows, const KvScan &sh)
{
    KvItem it{};
    it.s = sh.seq, it.h = sh.head, it.rt = sh.rt;
    kv_item_enter(a, tpi, few_rows, it);
    kv_item_tiles<TILE>(a, tpi, it.q, it.rt, &it);
    return it;
}

// What a CTA that gave up owes the counters, by one thread: the arrivals of its warps that
// have not told of their parts, and its own number, where it has not come to its join.
struct KvOwed {
    int joined, told[8];   // shared, zero at first
};
template <int TILE, int WARPS>
__device__ __noinline__ void kv_leave(const AttnArgs &a, int tpi, int few_rows, const KvScan &sh, const KvOwed &owed)
{
    const KvShare share(sh.total, sh.parts);
    const unsigned cta = sh.parts - 1 - blockIdx.x;
    unsigned long long u = share.start(cta);
    const unsigned long long u1 = share.start(cta + 1);
    KvItem it = kv_item_first<TILE>(a, tpi, few_rows, sh);
    int j0 = sh.off, told = 0;
    for (int w = 0; w < WARPS; ++w) told += owed.told[w];
    if (j0 > 0) atomicAdd(a.arrived + share.of(u - j0), WARPS - told);
    while (u1 - u > static_cast<unsigned>(it.n - j0)) {
        u += it.n - j0;
        j0 = 0;
        kv_item_next<TILE>(a, tpi, few_rows, it);
    }
    if (!owed.joined && j0 == 0 && u1 - u < static_cast<unsigned>(it.n))
        atomicSub(a.arrived + cta, WARPS * static_cast<int>(share.of(u + it.n - 1) - cta));
}

// True when V is finite in the positions [j0, j1) of a head (those of pages that are none
// count as that), by the whole warp.
template <int HD, class E>
__device__ __forceinline__ bool kv_finite(const AttnArgs &a, int s, int h, int j0, int j1)
{
    constexpr int LR = HD / 8, RW = 32 / LR, U = 4;
    const int lane = threadIdx.x & 31, grp = lane / LR;
    const E *vp = static_cast<const E *>(a.c.v) + lane % LR * 8;
    float nil = 0.f;
    for (int j = j0; j < j1; j += 32) {
        const long long at = j + lane < j1 ? kv_at(a.b, a.c, s, j + lane, h, nullptr) : -1;
#pragma unroll 1
        for (int k0 = 0; k0 < 32; k0 += U * RW) {
            float v[U][8];
            bool on[U];
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const long long va = __shfl_sync(0xFFFFFFFFu, at, k0 + u * RW + grp);
                on[u] = va >= 0;
                kv_load8(vp + (va < 0 ? 0 : va), v[u]);
            }
#pragma unroll
            for (int u = 0; u < U; ++u)
#pragma unroll
                for (int d = 0; d < 8; ++d) nil = on[u] ? fmaf(v[u][d], 0.f, nil) : nil;
        }
    }
    return !__any_sync(0xFFFFFFFFu, !(nil == 0.f));
}

// The chunk kernels' rows that are not finite, a warp's: they wait until its last item is out.
// In the loop over the items a call from here cost a long prompt 3 % without being made, and
// while a warp was at it the CTA's others would sit in bounded waits.
// Two things lead here: what a row sees, and 0 times what its tiles hold besides.  The
// second needs a V that is not finite where the tiles pass the rows' ends or the window:
// LOOK looks there, and where there is none the rows stay as they are: 3000 bf16 tokens of 8
// heads whose first V is NaN take 92 us, 62 without (5.0 ms with every row done again, 66 a
// position at a time).  Not for operands in parts, to which an infinity is NaN.
struct KvAgain {   // shared, n and must zero at first
    static constexpr int CAP = 4;
    int n;      // past CAP: all rows of the CTA's items
    int must;   // an item has a page outside the pool
    struct {
        unsigned rows;
        int t0, s, h, must;   // the row group's first token
    } rec[CAP];
    __device__ __forceinline__ void add(unsigned rows, int t0, int s, int h, bool bad)   // one thread
    {
        if (n < CAP) rec[n] = {rows, t0, s, h, bad};
        ++n;
        must |= bad;
    }
};
// lists: of the warps from warp0 on, four to a row group of tpt tokens.
template <int HD, class I, class E, int TILE, bool LOOK>
__device__ __noinline__ void kv_again(const AttnArgs &a, const KvAgain *lists, int warp0, int tpt, int tpi, int few_rows, const KvScan &sh)
{
    const int w = (threadIdx.x >> 5) - warp0, tok0 = (w >> 2) * tpt;
    const int r = (w & 3) * 32 + (threadIdx.x & 31), tok_in = r / a.group, hh = r - tok_in * a.group;
    const KvAgain &todo = lists[w];
    // rows of row tile rt of sequence s, head h, the lane's at position pos
    auto again = [&](unsigned rows, int s, int h, const KvSeq &q, int rt, int tok, bool must) {
        if (!rows) return;
        const int pos = q.len - q.n + tok;
        if (LOOK && !must) {
            KvItem it;
            kv_item_tiles<TILE>(a, tpi, q, rt, &it);
            const int low = __shfl_sync(0xFFFFFFFFu, pos, __ffs(rows) - 1), high = __shfl_sync(0xFFFFFFFFu, pos, 31 - __clz(rows));
            const int end = min(q.len, ((q.len - q.n + it.t1 - 1) / TILE + 1) * TILE);
            const KvSpan s0 = kv_span(low, a.window, a.sinks), s1 = kv_span(high, a.window, a.sinks);
            // past the first row's position, and between the first tokens and the last row's window
            if (kv_finite<HD, E>(a, s, h, low + 1, end) && kv_finite<HD, E>(a, s, h, s0.first, min(s1.lo, it.ns * TILE)) &&
                kv_finite<HD, E>(a, s, h, max(s0.first, it.lo * TILE), s1.lo))
                return;
        }
        kv_rows_again<HD, I, E>(a, rows, q.row0 + tok, h * a.group + hh, pos, s, h);
    };
    if (todo.n <= KvAgain::CAP) {
        for (int k = 0; k < todo.n; ++k) {
            const auto &x = todo.rec[k];
            KvSeq q;
            kv_seq(a.b, a.c, x.s, q, nullptr);
            again(x.rows, x.s, x.h, q, x.t0 / tpi, x.t0 + tok_in, x.must);
        }
        return;
    }
    const KvShare share(sh.total, sh.parts);
    const unsigned cta = sh.parts - 1 - blockIdx.x;
    const unsigned long long u1 = share.start(cta + 1);
    KvItem it = kv_item_first<TILE>(a, tpi, few_rows, sh);
    int j0 = sh.off;
    for (unsigned long long u = share.start(cta);;) {
        const int tok = it.t0 + tok0 + tok_in;
        const unsigned rows = __ballot_sync(0xFFFFFFFFu, j0 == 0 && tok_in < tpt && tok < it.t1);
        again(rows, it.s, it.h, it.q, it.rt, tok, todo.must);
        u += it.n - j0;
        if (u >= u1) break;
        j0 = 0;
        kv_item_next<TILE>(a, tpi, few_rows, it);
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
