// tb_kvtf32.cu — attention of chunks of new tokens over the paged cache to fp32
// accuracy on the 5th-generation tensor cores (include/tb_gguf_dequant.h part 4):
// k_kv_tf32, where k_kv_many does not apply: fp32 activations over any cache, 16-bit
// activations over a cache of another type, scales that are not positive.
//
// Items, units and the joining of parts are those of k_kv_many (tb_kvattn.cuh) with
// 128 query rows and tiles of 64 positions.  An fp32 operand x is hi + lo, both tf32
// (split_tf32: 2^-21 of x is lost), and a product is hi hi + hi lo + lo hi; a 16-bit
// cache is exact in tf32 and has no lo, and neither have 16-bit queries.
//
// Inside a CTA (512 threads, one CTA per SM):
//   warps 0-3   softmax, one row a thread; at an item's start Q into TMEM, in parts;
//   warps 4-7   the sums of P V, one row a thread, in registers: each tile's product
//               comes out of TMEM and is added with the factor of its running maximum;
//               epilogue and joining;
//   warps 8-11  operands: K in parts, V transposed (so that positions, the product's K,
//               are contiguous) and in parts, from the raw tiles to shared memory;
//   warp 12     the MMAs, A (Q, P) from TMEM, B (K, V) from shared memory;
//   warp 13     Q of the CTA's items to L2;
//   warps 14,15 K and V tiles by TMA, page by page.
// TMEM: Q's parts (2 x 128 columns), S (hi hi and, apart, the small products: 2 x 64;
// P's parts overwrite them), O (128).  Every tile's O is summed outside the tensor core,
// whose own sums would be chains over the whole context: fp32's accuracy would be
// lost in them.  An MMA of 64 columns was measured to take as long as one of 128, so
// Q_hi K_hi and Q_hi K_lo are one product, and O is one of all its dimensions.
//
// Measured (32 query and 8 kv heads of 128): 512 fp32 tokens at 1024 over an fp32 cache
// in 61 us, over a bf16 cache in 52; two times 2048 fp32 tokens from the start in 467 us,
// 147 TFLOP/s of the pairs that are seen, three tf32 products each.  A unit takes some
// 7000 cycles: 3600 from the last P to the next S (56 MMAs of 56 cycles, the tensor pipe),
// 2900 for the softmax between them.  To overlap the two takes a second S, and TMEM is
// full: S and O of 64 columns beside P, as was tried, make 96 MMAs of the 56 and came out
// slower (560 us against 530 then).
#include "tb_kvattn.cuh"

namespace tb {

static constexpr int kTfTile = 64;      // positions of a tile
static constexpr int kTfThreads = 512;
static constexpr int kTfMin = 4;        // units of a CTA, at least: 64 rows at 4096 take 63 us; with 2 74, with 8 55,
                                        // but 32 tokens of 16 heads at 512 then 24, not 20

struct TfArgs {
    AttnArgs a;
    int tpi;         // tokens of an item: 128 / G
    int few_rows;    // sequences of at most this many rows are another launch's
    int box;         // positions of one K or V box
};

struct TfShared {
    uint64_t kfull, kfree, vfull, vfree, kready, vready, qready, sfull, pready[2], ofull, oempty, done, join;
    KvScan scan;
    uint32_t tmem;
    int fail, bad[8];        // bad: i + 1 at place i % 8 for an item i of the CTA with a page outside the pool (K and V
                             // run at most 3 items ahead of the epilogue)
    KvOwed owed;
    KvAgain again[4];
    float corr[2][128];      // a tile's factor of the rows' sums so far
    float fin[2][2][128];    // an item's m and l
};

template <int HD, int TI, int TC>
struct TfCfg {
    static constexpr bool X32 = TC == QT_F32, QLO = TI == QT_F32;   // operands with a low part: K and V, Q
    static constexpr int RAW = kTfTile * HD * (X32 ? 4 : 2);        // K or V of a tile as it comes
    static constexpr int OP = kTfTile * HD * 4;                     // one part of it as an operand
    static constexpr int STAGE = 2048;                              // a warp's staging of rows of Q or O: [32][16] fp32
    static constexpr int SMEM = 1024 + 2 * RAW + (X32 ? 4 : 2) * OP + 8 * STAGE + static_cast<int>(sizeof(TfShared));
    static constexpr int PART = 128 * HD + 256;                     // floats of a partial result: O, m, l
};

// D[tmem] (+)= A[tmem] * B[smem desc]^T, tf32 operands, one thread
__device__ __forceinline__ void umma_tf32_ts(uint32_t d_tmem, uint32_t a_tmem, uint64_t b_desc, uint32_t idesc, uint32_t accumulate)
{
    asm volatile("{\n\t.reg .pred p;\n\t"
                 "setp.ne.b32 p, %4, 0;\n\t"
                 "tcgen05.mma.cta_group::1.kind::tf32 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d_tmem),
                 "r"(a_tmem), "l"(b_desc), "r"(idesc), "r"(accumulate)
                 : "memory");
}
__device__ __forceinline__ void sts_u128(uint32_t at, uint32_t a, uint32_t b, uint32_t c, uint32_t d)
{
    asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(at), "r"(a), "r"(b), "r"(c), "r"(d) : "memory");
}
__device__ __forceinline__ uint4 lds_raw(uint32_t at)   // in order with the barriers
{
    uint4 v;
    asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(at) : "memory");
    return v;
}
template <int TC>
__device__ __forceinline__ void widen2(uint32_t w, uint32_t &lo, uint32_t &hi)   // two 16-bit elements as fp32
{
    if constexpr (TC == QT_BF16) {
        lo = w << 16;
        hi = w & 0xFFFF0000u;
    } else {
        const float2 f = __half22float2(*reinterpret_cast<const __half2 *>(&w));
        lo = __float_as_uint(f.x);
        hi = __float_as_uint(f.y);
    }
}

// Where 4 floats of a row lie in a warp's staging: 16-byte pieces turned, so that 8 lanes
// meet 8 groups of banks whether they hold 8 rows or 2 rows' pieces.
__device__ __forceinline__ uint32_t tf_stage(int row, int piece) { return row * 64 + ((piece ^ ((row >> 1) & 3)) << 4); }
__device__ __forceinline__ float4 tf_load4(const float *p) { return *reinterpret_cast<const float4 *>(p); }
template <class I>
__device__ __forceinline__ float4 tf_load4(const I *p)
{
    const uint2 w = *reinterpret_cast<const uint2 *>(p);
    const I *x = reinterpret_cast<const I *>(&w);
    return make_float4(kv_f(x[0]), kv_f(x[1]), kv_f(x[2]), kv_f(x[3]));
}
__device__ __forceinline__ void tf_store4(float *p, const uint4 &v) { *reinterpret_cast<uint4 *>(p) = v; }
template <class I>
__device__ __forceinline__ void tf_store4(I *p, const uint4 &v)
{
    uint2 w;
    I *x = reinterpret_cast<I *>(&w);
    kv_store1(x, __uint_as_float(v.x));
    kv_store1(x + 1, __uint_as_float(v.y));
    kv_store1(x + 2, __uint_as_float(v.z));
    kv_store1(x + 3, __uint_as_float(v.w));
    *reinterpret_cast<uint2 *>(p) = w;
}
__device__ __forceinline__ void tf_add(uint32_t *a, const uint32_t *b)   // 32 sums
{
#pragma unroll
    for (int c = 0; c < 32; c += 2) {
        const float2 x = __fadd2_rn(make_float2(__uint_as_float(a[c]), __uint_as_float(a[c + 1])),
                                    make_float2(__uint_as_float(b[c]), __uint_as_float(b[c + 1])));
        a[c] = __float_as_uint(x.x), a[c + 1] = __float_as_uint(x.y);
    }
}

template <int HD, int TI, int TC>
__global__ void __launch_bounds__(kTfThreads, 1)
    k_kv_tf32(const __grid_constant__ CUtensorMap kmap, const __grid_constant__ CUtensorMap vmap,
              const __grid_constant__ TfArgs a)
{
    using Cfg = TfCfg<HD, TI, TC>;
    using I = typename KvType<TI>::E;
    using E = typename KvType<TC>::E;
    constexpr bool X32 = Cfg::X32, QLO = Cfg::QLO;
    constexpr int ES = X32 ? 4 : 2, RCB = HD * ES / 128;       // 128-byte columns of a raw tile
    // bytes of a 128-byte column of a raw tile, of K as an operand (high parts, then low ones:
    // together the 128 rows of one product), of V transposed
    constexpr uint32_t kCol = kTfTile * 128, kKCol = (X32 ? 2 : 1) * kCol, kVCol = HD * 128;
    constexpr int TQ = 0, TS = 256, TO = 384;                  // TMEM columns: Q's parts, S's or P's, O
    extern __shared__ __align__(1024) uint8_t smraw[];
    uint8_t *sm = reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(smraw) + 1023) & ~uintptr_t(1023));
    const uint32_t kraw = smem_u32(sm), vraw = kraw + Cfg::RAW, kop = vraw + Cfg::RAW, vhi = kop + (X32 ? 2 : 1) * Cfg::OP,
                   vlo = vhi + Cfg::OP;   // the last: fp32 caches
    uint8_t *stage = sm + 2 * Cfg::RAW + (X32 ? 4 : 2) * Cfg::OP;
    TfShared &sh = *reinterpret_cast<TfShared *>(stage + 8 * Cfg::STAGE);
    const int tid = threadIdx.x, lane = tid & 31, warp = __shfl_sync(0xFFFFFFFFu, tid >> 5, 0);
    const AttnArgs &aa = a.a;
    const uint32_t lim = aa.wait_limit;
    int *err = aa.err;

    if (tid == 0) {
        mbar_init(smem_u32(&sh.kfull), 1);
        mbar_init(smem_u32(&sh.vfull), 1);
        mbar_init(smem_u32(&sh.kfree), 128);
        mbar_init(smem_u32(&sh.vfree), 128);
        mbar_init(smem_u32(&sh.kready), 128);
        mbar_init(smem_u32(&sh.vready), 128);
        mbar_init(smem_u32(&sh.qready), 128);
        mbar_init(smem_u32(&sh.sfull), 1);
        mbar_init(smem_u32(&sh.pready[0]), 128);
        mbar_init(smem_u32(&sh.pready[1]), 128);
        mbar_init(smem_u32(&sh.ofull), 1);
        mbar_init(smem_u32(&sh.oempty), 128);
        mbar_init(smem_u32(&sh.done), 1);
        mbar_init(smem_u32(&sh.join), 128);
        fence_mbar_init();
        sh.fail = 0;
        for (int i = 0; i < 8; ++i) sh.bad[i] = 0;
        sh.owed = KvOwed{};
        for (int i = 0; i < 4; ++i) sh.again[i].n = sh.again[i].must = 0;
    }
    if (warp >= 14 && lane == 0) prefetch_map(warp == 15 ? &vmap : &kmap);
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    asm volatile("griddepcontrol.wait;" ::: "memory");
    KvCtaShare my;
    if (!kv_items_share<kTfTile, kTfMin, kTfThreads / 32, HD, I>(aa, a.tpi, a.few_rows, sh.scan, my)) return;
    if (warp == 12) {
        tmem_alloc(smem_u32(&sh.tmem), 512);
        tmem_relinquish();
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tm = sh.tmem;

    KvItem it = kv_item_first<kTfTile>(aa, a.tpi, a.few_rows, sh.scan);
    int j0 = sh.scan.off;        // the first of the item's tiles that is this CTA's
    unsigned long long u = my.u0;
    auto part_end = [&]() {      // the item's tiles [j0, part_end()) are this CTA's
        const unsigned long long left = my.u1 - u;
        return left < static_cast<unsigned>(it.n - j0) ? j0 + static_cast<int>(left) : it.n;
    };
    auto next_item = [&](int j1) {
        u += j1 - j0;
        j0 = 0;
        if (u < my.u1) kv_item_next<kTfTile>(aa, a.tpi, a.few_rows, it);
    };
    auto failed = [&]() { return *reinterpret_cast<volatile int *>(&sh.fail) != 0; };
    // A wait by a whole warp in step; false when the limit runs out or another role has given up.
    auto wait = [&](uint64_t *bar, uint32_t parity) {
        const uint32_t at = smem_u32(bar);
        for (uint32_t i = 0; i < lim; ++i) {
            if (__all_sync(0xFFFFFFFFu, mbar_try_wait(at, parity & 1u))) return true;
            if ((i & 15u) == 15u && __any_sync(0xFFFFFFFFu, failed())) break;
        }
        if (!failed()) atomicExch(err, ERR_WAIT_TIMEOUT);
        *reinterpret_cast<volatile int *>(&sh.fail) = 1;
        __syncwarp();
        return false;
    };

    uint32_t issued = 0;   // in the warps that copy
    bool ok = true;
    if (warp >= 12) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 80;");
        if (warp >= 14) {
            // ---- K (warp 14) and V tiles (15) as they are ----
            const bool kv = warp == 15;
            const uint32_t bar = smem_u32(kv ? &sh.vfull : &sh.kfull), raw = kv ? vraw : kraw;
            for (int item = 0; ok && u < my.u1; ++item) {
                const int j1 = part_end();
                for (int j = j0; ok && j < j1; ++j) {
                    const int p0 = kv_item_pos<kTfTile>(it, j), boxes = kTfTile / a.box;
                    // lane l: box l of the tile, its page (past the end, or seen by no row: one that reads as zeros)
                    int page = aa.c.n_pages, pos = 0;
                    const int p = p0 + lane * a.box;
                    if (lane < boxes && kv_item_sees(aa, it, p, a.box)) {
                        const uint32_t pi = fdiv(static_cast<uint32_t>(p), aa.c.page_div);
                        page = aa.b.pages[static_cast<long long>(it.s) * aa.b.pages_stride + pi];
                        pos = p - static_cast<int>(pi) * aa.c.page_size;
                        if (page < 0 || page >= aa.c.n_pages) {
                            atomicExch(err, ERR_RUNTIME);
                            *reinterpret_cast<volatile int *>(&sh.bad[item & 7]) = item + 1;
                            page = aa.c.n_pages;
                        }
                    }
                    const int y = aa.ax_pos == 0 ? pos : aa.ax_head == 0 ? it.h : page;
                    const int z = aa.ax_pos == 1 ? pos : aa.ax_head == 1 ? it.h : page;
                    const int w = aa.ax_pos == 2 ? pos : aa.ax_head == 2 ? it.h : page;
                    if (issued > 0) ok = wait(kv ? &sh.vfree : &sh.kfree, issued - 1u);
                    if (!ok) break;
                    if (lane == 0) mbar_expect_tx(bar, Cfg::RAW);
                    __syncwarp();
                    if (lane < boxes) {
                        const uint32_t dst = raw + lane * a.box * 128;
#pragma unroll
                        for (int cb = 0; cb < RCB; ++cb)
                            tma_load_4d(dst + cb * kCol, kv ? &vmap : &kmap, cb * (128 / ES), y, z, w, bar);
                    }
                    __syncwarp();
                    ++issued;
                }
                next_item(j1);
            }
        } else if (warp == 13) {
            // ---- Q of this CTA's items, from memory to L2 ----
            while (u < my.u1) {
                const int j1 = part_end();
                constexpr int ROW = HD * (TI == QT_F32 ? 4 : 2);
                for (int r = lane; r < (it.t1 - it.t0) * aa.group; r += 32) {
                    const int t = r / aa.group;
                    const char *p = reinterpret_cast<const char *>(static_cast<const I *>(aa.q.p) + (it.q.row0 + it.t0 + t) * aa.q.row +
                                                                   (it.h * aa.group + r - t * aa.group) * aa.q.head);
#pragma unroll
                    for (int b = 0; b < ROW; b += 128) asm volatile("prefetch.global.L2 [%0];" ::"l"(p + b));
                }
                next_item(j1);
            }
        } else if (warp == 12) {
            // ---- the MMAs: the whole warp in step, one lane issues ----
            constexpr uint32_t kFmt = (1u << 4) | (2u << 7) | (2u << 10) | (8u << 24);   // D fp32, A and B tf32, M = 128
            constexpr uint32_t id_s = kFmt | ((kTfTile >> 3) << 17), id_s2 = kFmt | ((2 * kTfTile >> 3) << 17),
                               id_o = kFmt | ((HD >> 3) << 17);
            const uint32_t tu = __shfl_sync(0xFFFFFFFFu, tm, 0);
            const uint64_t kd = sw128_desc(kop), vhd = sw128_desc(vhi), vld = sw128_desc(vlo);
            // D (+)= A B^T over K = 8 * steps; a column of B holds 32 of K
            auto product = [&](uint32_t d, uint32_t at, uint64_t b, uint32_t id, int steps, uint32_t col, bool first) {
#pragma unroll
                for (int ks = 0; ks < steps; ++ks)
                    umma_tf32_ts(d, at + ks * 8, b + (((ks >> 2) * col + (ks & 3) * 32) >> 4), id, (!first || ks > 0) ? 1u : 0u);
            };
            // the small products have columns of their own; those of Q's high part with both parts
            // of K are one product of 128 columns, which takes as long as one of 64
            auto issue_s = [&]() {
                product(tu + TS, tu + TQ, kd, X32 ? id_s2 : id_s, HD / 8, kKCol, true);
                if (QLO) product(tu + TS + kTfTile, tu + TQ + HD, kd, id_s, HD / 8, kKCol, !X32);
                umma_commit(smem_u32(&sh.sfull));
            };
            const uint32_t n_tiles = static_cast<uint32_t>(my.u1 - my.u0);
            uint32_t q = 0;
            int j1 = part_end(), left = j1 - j0;   // of the item's tiles, this one included
            ok = wait(&sh.qready, 0) && wait(&sh.kready, 0);
            if (ok) {
                tc_fence_after();
                if (elect_one()) issue_s();
                __syncwarp();
            }
            for (uint32_t n = 0; ok && n < n_tiles; ++n) {
                ok = wait(&sh.vready, n) && (n == 0 || wait(&sh.oempty, n - 1u)) && wait(&sh.pready[n & 1], n >> 1);
                if (!ok) break;
                tc_fence_after();
                if (elect_one()) {
                    if (X32) product(tu + TO, tu + TS, vld, id_o, kTfTile / 8, kVCol, true);
                    product(tu + TO, tu + TS + kTfTile, vhd, id_o, kTfTile / 8, kVCol, !X32);
                    product(tu + TO, tu + TS, vhd, id_o, kTfTile / 8, kVCol, false);
                    umma_commit(smem_u32(&sh.ofull));
                }
                __syncwarp();
                if (n + 1 == n_tiles) break;
                if (--left == 0) {   // the next item
                    next_item(j1);
                    j1 = part_end();
                    left = j1 - j0;
                    ok = wait(&sh.qready, ++q);
                }
                ok = ok && wait(&sh.kready, n + 1);
                if (!ok) break;
                tc_fence_after();
                if (elect_one()) issue_s();   // over P, in order after its product
                __syncwarp();
            }
            // every MMA issued is complete before TMEM is given back
            if (elect_one()) umma_commit(smem_u32(&sh.done));
            __syncwarp();
            mbar_wait_bounded(smem_u32(&sh.done), 0, err, kKvDrain);
        }
    } else if (warp >= 8) {
        // ---- operands: K in two parts, V transposed and in two parts ----
        asm volatile("setmaxnreg.dec.sync.aligned.u32 88;");
        const int tw = tid - 256;
        const uint32_t n_tiles = static_cast<uint32_t>(my.u1 - my.u0);
        auto split_k = [&](uint32_t n) {
            ok = ok && wait(&sh.kfull, n) && (n == 0 || wait(&sh.sfull, n - 1u));
            if (!ok) return;
            if constexpr (X32) {
#pragma unroll 1
                for (int i0 = 0; i0 < HD / 8; i0 += 8) {
                    const uint32_t at = static_cast<uint32_t>(i0 * 128 + tw) * 16u;
                    uint4 x[8];
#pragma unroll
                    for (int i = 0; i < 8; ++i) x[i] = lds_raw(kraw + at + i * 2048);
#pragma unroll
                    for (int i = 0; i < 8; ++i) {
                        uint4 h, l;
                        split_tf32(x[i].x, h.x, l.x);
                        split_tf32(x[i].y, h.y, l.y);
                        split_tf32(x[i].z, h.z, l.z);
                        split_tf32(x[i].w, h.w, l.w);
                        const uint32_t to = kop + at + i * 2048 + (i0 + i) / 4 * kCol;   // 2048 * 4: a raw column
                        sts_u128(to, h.x, h.y, h.z, h.w);
                        sts_u128(to + kCol, l.x, l.y, l.z, l.w);
                    }
                }
            } else {
                uint4 x[HD / 16];
#pragma unroll
                for (int i = 0; i < HD / 16; ++i) x[i] = lds_raw(kraw + static_cast<uint32_t>(i * 128 + tw) * 16u);
#pragma unroll
                for (int i = 0; i < HD / 16; ++i) {
                    const uint32_t c = i * 128 + tw, r = (c >> 3) & 63u, ch = (c & 7u) ^ (r & 7u);
                    const uint32_t d = (c >> 9) * 64 + ch * 8, oc = (d & 31u) >> 2;
                    uint32_t y[8];
                    widen2<TC>(x[i].x, y[0], y[1]);
                    widen2<TC>(x[i].y, y[2], y[3]);
                    widen2<TC>(x[i].z, y[4], y[5]);
                    widen2<TC>(x[i].w, y[6], y[7]);
                    const uint32_t to = kop + (d >> 5) * kKCol + r * 128;
                    sts_u128(to + ((oc ^ (r & 7u)) << 4), y[0], y[1], y[2], y[3]);
                    sts_u128(to + (((oc + 1) ^ (r & 7u)) << 4), y[4], y[5], y[6], y[7]);
                }
            }
            fence_proxy_async_smem();
            mbar_arrive(smem_u32(&sh.kfree));
            mbar_arrive(smem_u32(&sh.kready));
        };
        uint32_t n = 0;
        split_k(0);
        while (ok && u < my.u1) {
            const int j1 = part_end();
            for (int j = j0; j < j1; ++j, ++n) {
                ok = wait(&sh.vfull, n) && (n == 0 || wait(&sh.ofull, n - 1u));
                if (!ok) break;
                // 4 x 4 blocks; positions that there are not are zero: whatever V has there, 0 * it has to be 0
                const int rest = it.q.len - kv_item_pos<kTfTile>(it, j);
                const uint32_t pb = ((tw >> 5) << 2) | ((lane >> 1) & 3);
#pragma unroll 1
                for (int i0 = 0; i0 < HD / 32; i0 += 2) {
                    uint32_t xx[2][4][4];
#pragma unroll
                    for (int i = 0; i < 2; ++i) {
                        const uint32_t db = (i0 + i) * 8 + ((lane >> 3) << 1) + (lane & 1);
                        uint32_t (&x)[4][4] = xx[i];
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            const uint32_t p = pb * 4 + e;
                            if constexpr (X32) {
                                const uint4 w = lds_raw(vraw + (db >> 3) * kCol + p * 128 + (((db & 7u) ^ (p & 7u)) << 4));
                                x[e][0] = w.x, x[e][1] = w.y, x[e][2] = w.z, x[e][3] = w.w;
                            } else {
                                uint2 w;
                                const uint32_t at = vraw + (db >> 4) * kCol + p * 128 + ((((db >> 1) & 7u) ^ (p & 7u)) << 4) + (db & 1u) * 8;
                                asm volatile("ld.shared.v2.b32 {%0, %1}, [%2];" : "=r"(w.x), "=r"(w.y) : "r"(at) : "memory");
                                widen2<TC>(w.x, x[e][0], x[e][1]);
                                widen2<TC>(w.y, x[e][2], x[e][3]);
                            }
                        }
                    }
#pragma unroll
                    for (int i = 0; i < 2; ++i) {
                        const uint32_t db = (i0 + i) * 8 + ((lane >> 3) << 1) + (lane & 1);
                        uint32_t (&x)[4][4] = xx[i];
#pragma unroll
                        for (int e = 0; e < 4; ++e)
                            if (static_cast<int>(pb) * 4 + e >= rest) x[e][0] = x[e][1] = x[e][2] = x[e][3] = 0u;
#pragma unroll
                        for (int k = 0; k < 4; ++k) {
                            const uint32_t d = db * 4 + k, at = (pb >> 3) * kVCol + d * 128 + (((pb & 7u) ^ (d & 7u)) << 4);
                            if constexpr (X32) {
                                uint32_t h[4], l[4];
#pragma unroll
                                for (int e = 0; e < 4; ++e) split_tf32(x[e][k], h[e], l[e]);
                                sts_u128(vhi + at, h[0], h[1], h[2], h[3]);
                                sts_u128(vlo + at, l[0], l[1], l[2], l[3]);
                            } else {
                                sts_u128(vhi + at, x[0][k], x[1][k], x[2][k], x[3][k]);
                            }
                        }
                    }
                }
                fence_proxy_async_smem();
                mbar_arrive(smem_u32(&sh.vfree));
                mbar_arrive(smem_u32(&sh.vready));
                if (n + 1 < n_tiles) split_k(n + 1);
                if (!ok) break;
            }
            next_item(j1);
        }
    } else if (warp < 4) {
        // ---- softmax: thread = row ----
        asm volatile("setmaxnreg.inc.sync.aligned.u32 160;");
        const uint32_t lanes = static_cast<uint32_t>(warp * 32) << 16;
        const uint32_t tq = tm + TQ + lanes, ts = tm + TS + lanes;
        const uint32_t mine = smem_u32(stage + warp * Cfg::STAGE);
        const int tok_in = tid / aa.group, hh = tid - tok_in * aa.group;
        const float sc = aa.scale2;
        uint32_t cnt = 0, items = 0;
        while (ok && u < my.u1) {
            const int j1 = part_end();
            const int tok = it.t0 + tok_in;
            const bool on = tok_in < a.tpi && tok < it.t1;
            const int p0 = it.q.len - it.q.n, pos = on ? p0 + tok : -1, pmin = p0 + it.t0, pmax = p0 + it.t1 - 1;
            // Q (the products with the last one are complete: their S has been read)
            // 8 rows of 16 dimensions a load, through shared memory to a row a thread
            const long long off = on ? (it.q.row0 + tok) * aa.q.row + (it.h * aa.group + hh) * aa.q.head : -1;
            long long ro[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) ro[i] = __shfl_sync(0xFFFFFFFFu, off, i * 8 + (lane >> 2));
#pragma unroll 1
            for (int c = 0; c < HD; c += 64) {
                float4 y[4][4];
#pragma unroll
                for (int k = 0; k < 4; ++k)
#pragma unroll
                    for (int i = 0; i < 4; ++i)
                        y[k][i] = ro[i] >= 0 ? tf_load4(static_cast<const I *>(aa.q.p) + ro[i] + c + k * 16 + (lane & 3) * 4)
                                             : make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
                for (int k = 0; k < 4; k += 2) {
                    uint32_t h[32], l[32];
#pragma unroll
                    for (int k2 = 0; k2 < 2; ++k2) {
                        __syncwarp();
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            const float4 v = y[k + k2][i];
                            sts_u128(mine + tf_stage(i * 8 + (lane >> 2), lane & 3), __float_as_uint(v.x), __float_as_uint(v.y),
                                     __float_as_uint(v.z), __float_as_uint(v.w));
                        }
                        __syncwarp();
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            const uint4 v = lds_raw(mine + tf_stage(lane, i));
                            const int e = k2 * 16 + i * 4;
                            split_tf32(v.x, h[e], l[e]);
                            split_tf32(v.y, h[e + 1], l[e + 1]);
                            split_tf32(v.z, h[e + 2], l[e + 2]);
                            split_tf32(v.w, h[e + 3], l[e + 3]);
                        }
                    }
                    tmem_st32(tq + c + k * 16, h);
                    if (QLO) tmem_st32(tq + HD + c + k * 16, l);
                }
            }
            tmem_wait_st();
            tc_fence_before();
            mbar_arrive(smem_u32(&sh.qready));
            float m = -INFINITY, l = 0.f;
            for (int j = j0; j < j1; ++j, ++cnt) {
                ok = wait(&sh.sfull, cnt);
                if (!ok) break;
                tc_fence_after();
                uint32_t s[64], t[32];
                tmem_ld32(ts, s);
                if (QLO || X32) tmem_ld32(ts + 64, t);
                tmem_ld32(ts + 32, s + 32);
                tmem_wait_ld(s);
                after_wait(s + 32);
                if constexpr (QLO || X32) {
                    after_wait(t);
                    uint32_t r[32];
                    tmem_ld32(ts + 96, r);
                    tf_add(s, t);
                    tmem_wait_ld(r);
                    tf_add(s + 32, r);
                }
#pragma unroll
                for (int c = 0; c < 64; c += 2) {
                    const float2 x = __ffma2_rn(make_float2(__uint_as_float(s[c]), __uint_as_float(s[c + 1])),
                                                make_float2(sc, sc), make_float2(0.f, 0.f));
                    s[c] = __float_as_uint(x.x), s[c + 1] = __float_as_uint(x.y);
                }
                const int k0 = kv_item_pos<kTfTile>(it, j);
                if (k0 + kTfTile - 1 > pmin) {
                    const int last = pos - k0;   // the last column that the row sees
#pragma unroll
                    for (int c = 0; c < 64; ++c)
                        if (c > last) s[c] = 0xFF800000u;
                }
                if (aa.window > 0 && k0 <= pmax - aa.window && k0 + kTfTile > aa.sinks) {
                    const int first = pos - aa.window + 1 - k0, sinks = aa.sinks - k0;   // columns below first, past the sinks
#pragma unroll
                    for (int c = 0; c < 64; ++c)
                        if (c < first && c >= sinks) s[c] = 0xFF800000u;
                }
                float mxs[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
                for (int c = 0; c < 64; c += 2)
                    mxs[(c >> 1) & 3] = fmaxf(fmaxf(__uint_as_float(s[c]), __uint_as_float(s[c + 1])), mxs[(c >> 1) & 3]);
                const float mx = fmaxf(fmaxf(mxs[0], mxs[1]), fmaxf(mxs[2], mxs[3]));
                float corr = 1.f;
                if (__any_sync(0xFFFFFFFFu, on && mx > m + 8.f)) {
                    const float mn = fmaxf(m, mx);
                    corr = m == -INFINITY ? 0.f : ex2(m - mn);
                    l *= corr;
                    m = mn;
                }
                sh.corr[cnt & 1][tid] = corr;
                const float nm = m == -INFINITY ? 0.f : -m;
                const float2 nm2 = make_float2(nm, nm), neg = make_float2(-1.f, -1.f);
                float2 sum[2] = {make_float2(0.f, 0.f), make_float2(0.f, 0.f)};
#pragma unroll
                for (int h = 0; h < 2; ++h) {
#pragma unroll
                    for (int c = 0; c < 32; c += 2) {
                        uint32_t *y = s + h * 32 + c;
                        float2 x = __fadd2_rn(make_float2(__uint_as_float(y[0]), __uint_as_float(y[1])), nm2);
                        x.x = ex2(x.x);
                        x.y = ex2(x.y);
                        sum[(c >> 1) & 1] = __fadd2_rn(sum[(c >> 1) & 1], x);
                        y[0] = (__float_as_uint(x.x) + 0x1000u) & 0xFFFFE000u;   // as split_tf32
                        y[1] = (__float_as_uint(x.y) + 0x1000u) & 0xFFFFE000u;
                        x = __ffma2_rn(make_float2(__uint_as_float(y[0]), __uint_as_float(y[1])), neg, x);
                        t[c] = __float_as_uint(x.x), t[c + 1] = __float_as_uint(x.y);
                    }
                    tmem_st32(ts + h * 32, s + h * 32);
                    tmem_st32(ts + kTfTile + h * 32, t);
                }
                l += (sum[0].x + sum[0].y) + (sum[1].x + sum[1].y);
                if (j == j1 - 1) sh.fin[items & 1][0][tid] = m, sh.fin[items & 1][1][tid] = l;
                tmem_wait_st();
                tc_fence_before();
                mbar_arrive(smem_u32(&sh.pready[cnt & 1]));
            }
            ++items;
            next_item(j1);
        }
    } else {
        // ---- the sums of P V, in registers: thread = row ----
        asm volatile("setmaxnreg.inc.sync.aligned.u32 184;");
        const int row = tid - 128;
        const uint32_t mine = smem_u32(stage + warp * Cfg::STAGE);
        const uint32_t to = tm + TO + (static_cast<uint32_t>((warp & 3) * 32) << 16);
        const int tok_in = row / aa.group, hh = row - tok_in * aa.group;
        uint32_t cnt = 0, items = 0, joins = 0;
        int tell = -1;   // the CTA that waits for this one's part
        auto told = [&]() {   // each warp for its rows
            kv_arrive(aa, tell);
            sh.owed.told[warp - 4] = 1;
            tell = -1;
        };
        while (ok && u < my.u1) {
            const int j1 = part_end();
            const int tok = it.t0 + tok_in;
            const bool on = tok_in < a.tpi && tok < it.t1;
            float O[HD], m = -INFINITY, l = 0.f;
#pragma unroll
            for (int d = 0; d < HD; ++d) O[d] = 0.f;
            for (int j = j0; j < j1; ++j, ++cnt) {
                ok = wait(&sh.ofull, cnt) && wait(&sh.pready[cnt & 1], cnt >> 1);
                if (!ok) break;
                tc_fence_after();
                const float corr = sh.corr[cnt & 1][row];
                if (j == j1 - 1) m = sh.fin[items & 1][0][row], l = sh.fin[items & 1][1][row];
#pragma unroll
                for (int c = 0; c < HD; c += 32) {
                    uint32_t o[32];
                    tmem_ld32(to + c, o);
                    tmem_wait_ld(o);
                    if (c + 32 == HD) {
                        tc_fence_before();
                        mbar_arrive(smem_u32(&sh.oempty));
                    }
#pragma unroll
                    for (int i = 0; i < 32; ++i) O[c + i] = fmaf(O[c + i], corr, __uint_as_float(o[i]));
                }
                if (tell >= 0) told();
            }
            if (!ok) break;
            const bool bad = *reinterpret_cast<volatile int *>(&sh.bad[items & 7]) == static_cast<int>(items) + 1;
            if (j0 > 0) {
                // ---- not the item's beginning: the part goes to the CTA that has it
                // (a page outside the pool: as NaN, so that the rows are done again there) ----
                float4 *part = reinterpret_cast<float4 *>(aa.part + static_cast<size_t>(my.cta) * Cfg::PART) + row;
                if (on) {   // rows that there are not stay out of the traffic
#pragma unroll
                    for (int c = 0; c < HD; c += 4) __stcg(part + c / 4 * 128, make_float4(O[c], O[c + 1], O[c + 2], O[c + 3]));
                    float2 *ml = reinterpret_cast<float2 *>(aa.part + static_cast<size_t>(my.cta) * Cfg::PART + 128 * HD) + row;
                    __stcg(ml, make_float2(m, bad ? NAN : l));
                }
                tell = static_cast<int>(my.share.of(u - j0));
            } else {
                // ---- the beginning: the other parts, of the CTAs after this one, in order (waited
                // for, as every wait, within a limit: those CTAs were started before this one) ----
                bool odd = bad;
                if (j1 < it.n) {
                    const unsigned others = my.share.of(u + it.n - 1) - my.cta;
                    if (row == 0) {
                        if (!kv_await(aa, my.cta, 4 * others, failed)) {
                            if (!failed()) atomicExch(err, ERR_WAIT_TIMEOUT);
                            *reinterpret_cast<volatile int *>(&sh.fail) = 1;
                        }
                        sh.owed.joined = 1;
                    }
                    __syncwarp();
                    mbar_arrive(smem_u32(&sh.join));
                    ok = wait(&sh.join, joins++);
                    if (!ok) break;
                    for (unsigned c = 0; c < others && on; ++c) {
                        const float *pp = aa.part + static_cast<size_t>(my.cta + 1 + c) * Cfg::PART;
                        const float2 ml = __ldcg(reinterpret_cast<const float2 *>(pp + 128 * HD) + row);
                        const float mx = fmaxf(m, ml.x);
                        const float f0 = m == -INFINITY ? 0.f : ex2(m - mx), f1 = ml.x == -INFINITY ? 0.f : ex2(ml.x - mx);
                        // nothing seen: l is 0, unless what was seen was NaN
                        l = (m == -INFINITY ? l : l * f0) + (ml.x == -INFINITY ? ml.y : ml.y * f1);
                        m = mx;
                        const float4 *p4 = reinterpret_cast<const float4 *>(pp) + row;
#pragma unroll
                        for (int d = 0; d < HD; d += 4) {
                            const float4 v = __ldcg(p4 + d / 4 * 128);
                            O[d] = O[d] * f0 + v.x * f1;
                            O[d + 1] = O[d + 1] * f0 + v.y * f1;
                            O[d + 2] = O[d + 2] * f0 + v.z * f1;
                            O[d + 3] = O[d + 3] * f0 + v.w * f1;
                        }
                    }
                }
                I *out = static_cast<I *>(const_cast<void *>(aa.o.p));
                const long long grow = static_cast<long long>(it.q.row0) + tok;
                const int ghead = it.h * aa.group + hh;
                const float inv = l == 0.f ? 0.f : 1.0f / l;
                odd = odd || !isfinite(l) || m == INFINITY;
                float nil = 0.f;   // stays zero where everything is finite
#pragma unroll
                for (int d = 0; d < HD; ++d) nil = fmaf(O[d], 0.f, nil);
                odd = odd || !(nil == 0.f);
                const long long off = on ? grow * aa.o.row + ghead * aa.o.head : -1;
                long long ro[4];
#pragma unroll
                for (int i = 0; i < 4; ++i) ro[i] = __shfl_sync(0xFFFFFFFFu, off, i * 8 + (lane >> 2));
#pragma unroll
                for (int d = 0; d < HD; d += 16) {   // through shared memory: 8 rows of 16 dimensions a store
                    __syncwarp();
#pragma unroll
                    for (int i = 0; i < 4; ++i)
                        sts_u128(mine + tf_stage(lane, i), __float_as_uint(O[d + i * 4] * inv), __float_as_uint(O[d + i * 4 + 1] * inv),
                                 __float_as_uint(O[d + i * 4 + 2] * inv), __float_as_uint(O[d + i * 4 + 3] * inv));
                    __syncwarp();
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const uint4 v = lds_raw(mine + tf_stage(i * 8 + (lane >> 2), lane & 3));
                        if (ro[i] >= 0) tf_store4(out + ro[i] + d + (lane & 3) * 4, v);
                    }
                }
                // rows that are not finite: V of a position that a row does not see may have been
                // (0 * NaN), or a page lies outside the pool.  Once more at the end, over their own positions only.
                __syncwarp();
                const unsigned rows = __ballot_sync(0xFFFFFFFFu, odd && on);
                if (rows && lane == 0) sh.again[warp - 4].add(rows, it.t0, it.s, it.h, true);
            }
            ++items;
            next_item(j1);
        }
        if (tell >= 0) told();
        __syncwarp();
        if (sh.again[warp - 4].n > 0) kv_again<HD, I, E, kTfTile, false>(aa, sh.again, 4, a.tpi, a.tpi, a.few_rows, sh.scan);
    }
    // ---- the end: nothing in flight, TMEM given back ----
    tc_fence_before();
    __syncthreads();
    // a wait ran out: the counters, and the copies still in flight
    if (sh.fail && tid == 0) kv_leave<kTfTile, 4>(aa, a.tpi, a.few_rows, sh.scan, sh.owed);
    if (sh.fail && issued > 0)
        mbar_wait_bounded(smem_u32(warp == 15 ? &sh.vfull : &sh.kfull), (issued - 1) & 1u, nullptr, kKvDrain);
    __syncthreads();
    if (warp == 12) {
        tc_fence_after();
        tmem_dealloc(tm, 512);
    }
}

// ---------------------------------------------------------------------------
// host side
// ---------------------------------------------------------------------------
size_t kv_tf32_part_bytes() { return sizeof(float) * TfCfg<128, QT_F32, QT_F32>::PART; }

template <int HD, int TI, int TC>
static int tf_launch(TfArgs &w, int sms, cudaStream_t st)
{
    AttnArgs &a = w.a;
    CUtensorMap km, vm;
    int ax[3];
    w.box = kTfTile;
    while (a.c.page_size % w.box) w.box >>= 1;   // at least 16: it divides every page
    if (!kv_maps(a.c, HD, TC, w.box, &km, &vm, ax)) return 0;
    a.ax_pos = ax[0], a.ax_head = ax[1], a.ax_page = ax[2];
    auto fn = k_kv_tf32<HD, TI, TC>;
    if (!smem_attr_once(reinterpret_cast<const void *>(fn), TfCfg<HD, TI, TC>::SMEM)) {
        cudaGetLastError();
        return 0;
    }
    void *args[] = {&km, &vm, &w};
    return kv_launch(reinterpret_cast<const void *>(fn), dim3(sms < kManyCtas ? sms : kManyCtas), kTfThreads,
                     TfCfg<HD, TI, TC>::SMEM, args, st);
}

template <int HD, int TI>
static int tf_types(TfArgs &w, int tc, int sms, cudaStream_t st)
{
    return tc == QT_F32   ? tf_launch<HD, TI, QT_F32>(w, sms, st)
           : tc == QT_F16 ? tf_launch<HD, TI, QT_F16>(w, sms, st)
                          : tf_launch<HD, TI, QT_BF16>(w, sms, st);
}

template <int HD>
static int tf_hd(TfArgs &w, int ti, int tc, int sms, cudaStream_t st)
{
    return ti == QT_F32   ? tf_types<HD, QT_F32>(w, tc, sms, st)
           : ti == QT_F16 ? tf_types<HD, QT_F16>(w, tc, sms, st)
                          : tf_types<HD, QT_BF16>(w, tc, sms, st);
}

int kv_tf32_launch(AttnArgs a, int hd, int ti, int tc, int few_rows, int sms, cudaStream_t st)
{
    TfArgs w{a, 128 / a.group, few_rows, 0};
    return hd == 128 ? tf_hd<128>(w, ti, tc, sms, st) : tf_hd<64>(w, ti, tc, sms, st);
}

}  // namespace tb
