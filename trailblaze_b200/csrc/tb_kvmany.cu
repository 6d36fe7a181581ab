// tb_kvmany.cu — attention of chunks of new tokens over the paged cache on the
// 5th-generation tensor cores (include/tb_gguf_dequant.h part 4): k_kv_many, for
// 16-bit activations over a cache of the same type and enough query rows per kv
// head to fill tiles of 128.
//
// An item is (sequence, kv head, 2 x 128 query rows): with G query heads per kv
// head a group of 128 rows holds 128 / G whole tokens, row = token * G + head.  A
// unit is an item's product with a tile of 128 positions.  All items' units, laid
// end to end, are cut into equal parts, one per CTA (one CTA per SM): causal
// triangles, windows and ragged lengths balance by themselves, and a short chunk
// late in a long context still fills the GPU.  An item cut between CTAs is joined
// by the CTA that has its beginning, in CTA order, so results repeat bit for bit.
//
// Inside a CTA (384 threads):
//   warps 0-3, 4-7  softmax of row group 0 / 1, one row a thread;
//   warp 8          the MMAs, one elected thread: S_g = Q_g K^T (128 x 128, both
//                   operands in shared memory), O_g += P_g V (P_g read from TMEM);
//   warp 9          K and V tiles by TMA into a ring, page by page;
//   warp 10         Q tiles by TMA (the next item's while the last one's softmax
//                   and epilogue still run);
//   warp 11         zeros into V past a sequence's end.
// TMEM: S_0, S_1 (128 fp32 columns each, P_g overwrites the first half of S_g as
// 16-bit pairs), O_0, O_1.  The two groups take turns on the tensor core: while
// one's softmax runs, the other's products do.  The MMA order PV_g(j), S_g(j + 1)
// makes the overwriting of P_g safe without a barrier, since MMAs of one thread
// execute in order; when S_g(j) is complete so is PV_g(j - 1), which is why the
// softmax threads may rescale O_g between seeing S_g and handing over P_g.
//
// The running maximum moves only when a score passes it by 2^8, so rescaling O is
// rare.  P is rounded to the cache's type for the second product, whose unit takes
// nothing wider: 2^-9 (bf16) or 2^-12 (fp16) of each term, unbiased, about what the
// output's own rounding is; sums are fp32 of the unrounded P.  fp16 ends at 2^-24: its
// numerators lie 2^7 higher, up to 2^15, so that what it cannot hold lies 2^-32 below
// the largest.
//
// Measured (32 query and 8 kv heads of 128, bf16): 8192 tokens from the start in 559
// us, 983 TFLOP/s of the pairs that are seen (call after call under the power cap; 500
// to 510 us in a burst of 20); 512 tokens at 4096 in 46 us.  A unit
// takes some 3000 cycles, 2048 of them tensor pipe: what is left is the way from the
// last P over P V and the next S back to the softmax warps (1200) and their 128
// exponentials a row (1024 of the multi-function unit), which the other group's
// products cover in part.
#include "tb_kvattn.cuh"

namespace tb {

static constexpr int kTileN = 128;      // positions of a tile
static constexpr int kManyThreads = 384;
static constexpr int kManyMin = 3;      // units of a CTA, at least (16 tokens at 4096: 29 us; with 1: 62)

struct ManyArgs {
    AttnArgs a;
    int tpt, tpi;    // tokens of a row group, 128 / G, and of an item, twice that
    int few_rows;    // sequences of at most this many rows are another launch's
    int box;         // positions of one K or V box
    int bf16;
};

template <int HD>
struct ManyCfg {
    static constexpr int SLOT = kTileN * HD * 2;         // one K or V tile
    static constexpr int QG = 128 * HD * 2;              // one row group's Q
    static constexpr int NS = HD == 128 ? 4 : 8;         // ring slots
    static constexpr int STAGE = 4096;                   // a softmax warp's staging for its output rows
    static constexpr int SMEM = 1024 + 2 * QG + NS * SLOT + 8 * STAGE + 2048;
    static constexpr int PART = 256 * HD + 512;          // floats of a partial result: O, m, l
};

// What the MMA and softmax warps need of an item (this CTA's part of it), written
// by the Q warp with the item's Q.
struct alignas(16) ManyPart {
    int row0, len, n, t0;   // the sequence's first row, length and new tokens; the item's first token,
    int t1, s, h, tiles;    // its end; sequence, kv head; the item's position tiles,
    int ns, lo, j0, j1;     // where they lie, and this CTA's [j0, j1) of them
    unsigned peer, pad[3];  // j0 > 0: the CTA that joins the parts; else how many others there are
};

struct ManyShared {
    ManyPart part[4];
    uint64_t sfull[2], pready[2][2], ofull[2], qfull, qempty, done, join, kvfull[8], kvempty[4], vready[8];
    KvScan scan;
    uint32_t tmem;
    int fail, bad[8];       // bad: i + 1 at place i % 8 for an item i of the CTA with a page outside the pool (K and V
                            // run at most 5 items ahead of the epilogue)
    KvOwed owed;
    KvAgain again[8];
};
static_assert(sizeof(ManyShared) <= 2048, "ManyShared");

// D[tmem] (+)= A[tmem] * B[smem desc], one thread
__device__ __forceinline__ void umma_f16_ts(uint32_t d_tmem, uint32_t a_tmem, uint64_t b_desc, uint32_t idesc,
                                            uint32_t accumulate)
{
    asm volatile("{\n\t.reg .pred p;\n\t"
                 "setp.ne.b32 p, %4, 0;\n\t"
                 "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d_tmem),
                 "r"(a_tmem), "l"(b_desc), "r"(idesc), "r"(accumulate)
                 : "memory");
}
// Shared-memory descriptor of V as the B operand: rows are positions (the
// product's K), 128-byte columns of 64 dimensions (its N, "MN-major") with the
// 128-byte swizzle.  Leading byte offset: from one 64-dimension column to the
// next; stride byte offset: from 8 positions to the next 8.
__device__ __forceinline__ uint64_t v_desc(uint32_t saddr)
{
    uint64_t d = 0;
    d |= static_cast<uint64_t>((saddr >> 4) & 0x3FFFu);
    d |= static_cast<uint64_t>((kTileN * 128u) >> 4) << 16;
    d |= static_cast<uint64_t>(1024u >> 4) << 32;
    d |= static_cast<uint64_t>(1u) << 46;
    d |= static_cast<uint64_t>(2u) << 61;
    return d;
}
__device__ __forceinline__ void tma_load_3d(uint32_t dst, const CUtensorMap *map, int x, int y, int z, uint32_t bar)
{
    asm volatile("cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], "
                 "[%5];" ::"r"(dst),
                 "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(y), "r"(z), "r"(bar)
                 : "memory");
}

template <int HD, class I>
__global__ void __launch_bounds__(kManyThreads, 1)
    k_kv_many(const __grid_constant__ CUtensorMap qmap, const __grid_constant__ CUtensorMap kmap,
              const __grid_constant__ CUtensorMap vmap, const __grid_constant__ ManyArgs a)
{
    using Cfg = ManyCfg<HD>;
    constexpr int CB = HD / 64;   // 128-byte columns
    constexpr int NS = Cfg::NS;
    constexpr bool BF = std::is_same<I, __nv_bfloat16>::value;
    // m is moved when a score passes it by 2^TOP, to 2^UP below the largest score then
    constexpr float TOP = BF ? 8.f : 15.f, UP = BF ? 0.f : 7.f;
    extern __shared__ __align__(1024) uint8_t smraw[];
    uint8_t *sm = reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(smraw) + 1023) & ~uintptr_t(1023));
    uint8_t *stage = sm + 2 * Cfg::QG + NS * Cfg::SLOT;
    ManyShared &sh = *reinterpret_cast<ManyShared *>(stage + 8 * Cfg::STAGE);
    const uint32_t qbase = smem_u32(sm), ring = qbase + 2 * Cfg::QG;
    const int tid = threadIdx.x, lane = tid & 31, warp = __shfl_sync(0xFFFFFFFFu, tid >> 5, 0);
    const uint32_t lim = a.a.wait_limit;
    int *err = a.a.err;

    if (tid == 0) {
        for (int g = 0; g < 2; ++g) {
            mbar_init(smem_u32(&sh.sfull[g]), 1);
            mbar_init(smem_u32(&sh.pready[g][0]), 128);
            mbar_init(smem_u32(&sh.pready[g][1]), 128);
            mbar_init(smem_u32(&sh.ofull[g]), 1);
        }
        mbar_init(smem_u32(&sh.qfull), 1);
        mbar_init(smem_u32(&sh.qempty), 1);
        mbar_init(smem_u32(&sh.done), 1);
        mbar_init(smem_u32(&sh.join), 256);
        for (int i = 0; i < NS; ++i) {
            mbar_init(smem_u32(&sh.kvfull[i]), 1);
            if (i % 2 == 0) mbar_init(smem_u32(&sh.kvempty[i / 2]), 1);
            mbar_init(smem_u32(&sh.vready[i]), 1);
        }
        fence_mbar_init();
        sh.fail = 0;
        for (int i = 0; i < 8; ++i) sh.bad[i] = 0;
        sh.owed = KvOwed{};
        for (int i = 0; i < 8; ++i) sh.again[i].n = sh.again[i].must = 0;
    }
    if (warp == 9 && lane < 2) prefetch_map(lane ? &vmap : &kmap);
    if (warp == 10 && lane == 0) prefetch_map(&qmap);
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    asm volatile("griddepcontrol.wait;" ::: "memory");
    KvCtaShare my;
    if (!kv_items_share<kTileN, kManyMin, kManyThreads / 32, HD, I>(a.a, a.tpi, a.few_rows, sh.scan, my)) return;
    if (warp == 8) {
        tmem_alloc(smem_u32(&sh.tmem), 512);
        tmem_relinquish();
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tm = sh.tmem;

    KvItem it = kv_item_first<kTileN>(a.a, a.tpi, a.few_rows, sh.scan);
    int j0 = sh.scan.off;        // the first of the item's tiles that is this CTA's
    unsigned long long u = my.u0;
    // the item's tiles [j0, j1) are this CTA's
    auto part_end = [&]() {
        const unsigned long long left = my.u1 - u;
        return left < static_cast<unsigned>(it.n - j0) ? j0 + static_cast<int>(left) : it.n;
    };
    auto next_item = [&](int j1) {
        u += j1 - j0;
        j0 = 0;
        if (u < my.u1) kv_item_next<kTileN>(a.a, a.tpi, a.few_rows, it);
    };
    auto failed = [&]() { return *reinterpret_cast<volatile int *>(&sh.fail) != 0; };
    // Waits, by a whole warp in step, for one or two barriers; false when the limit runs
    // out or another role has given up.
    auto wait2 = [&](uint64_t *b0, uint32_t p0, uint64_t *b1, uint32_t p1) {
        const uint32_t at0 = smem_u32(b0), at1 = smem_u32(b1);
        for (uint32_t i = 0; i < lim; ++i) {
            const bool r0 = mbar_try_wait(at0, p0 & 1u), r1 = mbar_try_wait(at1, p1 & 1u);
            if (__all_sync(0xFFFFFFFFu, r0 && r1)) return true;
            if ((i & 15u) == 15u && __any_sync(0xFFFFFFFFu, failed())) break;
        }
        if (!failed()) atomicExch(err, ERR_WAIT_TIMEOUT);
        *reinterpret_cast<volatile int *>(&sh.fail) = 1;
        __syncwarp();
        return false;
    };
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

    uint32_t kv_issued = 0, q_issued = 0;   // in the warps that issue them
    if (warp >= 8) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 88;");
        if (warp == 9) {
            // ---- K and V ----
            bool ok = true;
            for (int item = 0; ok && u < my.u1; ++item) {
                const int j1 = part_end();
                for (int j = j0; ok && j < j1; ++j) {
                    const int p0 = kv_item_pos<kTileN>(it, j), boxes = kTileN / a.box;
                    // lane l: box l of the tile, its page (past the end, or seen by no row: one that reads as zeros)
                    int page = a.a.c.n_pages, pos = 0;
                    const int p = p0 + lane * a.box;
                    if (lane < boxes && kv_item_sees(a.a, it, p, a.box)) {
                        const uint32_t pi = fdiv(static_cast<uint32_t>(p), a.a.c.page_div);
                        page = a.a.b.pages[static_cast<long long>(it.s) * a.a.b.pages_stride + pi];
                        pos = p - static_cast<int>(pi) * a.a.c.page_size;
                        if (page < 0 || page >= a.a.c.n_pages) {
                            atomicExch(err, ERR_RUNTIME);
                            *reinterpret_cast<volatile int *>(&sh.bad[item & 7]) = item + 1;
                            page = a.a.c.n_pages;
                        }
                    }
                    const int y = a.a.ax_pos == 0 ? pos : a.a.ax_head == 0 ? it.h : page;
                    const int z = a.a.ax_pos == 1 ? pos : a.a.ax_head == 1 ? it.h : page;
                    const int w = a.a.ax_pos == 2 ? pos : a.a.ax_head == 2 ? it.h : page;
                    for (int kv = 0; kv < 2; ++kv) {
                        const uint32_t n = kv_issued, slot = n % NS, bar = smem_u32(&sh.kvfull[slot]);
                        if (n >= NS) ok = wait(&sh.kvempty[((n - NS + 1) / 2) % (NS / 2)], (n - NS + 1) / NS);
                        if (!ok) break;
                        if (lane == 0) mbar_expect_tx(bar, Cfg::SLOT);
                        __syncwarp();
                        if (lane < boxes) {
                            const uint32_t dst = ring + slot * Cfg::SLOT + lane * a.box * 128;
#pragma unroll
                            for (int cb = 0; cb < CB; ++cb)
                                tma_load_4d(dst + cb * kTileN * 128, kv ? &vmap : &kmap, cb * 64, y, z, w, bar);
                        }
                        __syncwarp();
                        ++kv_issued;
                    }
                }
                next_item(j1);
            }
        } else if (warp == 10) {
            // ---- Q ----
            bool ok = true;
            while (ok && u < my.u1) {
                const int j1 = part_end();
                if (q_issued > 0) ok = wait(&sh.qempty, q_issued - 1u);
                if (!ok) break;
                // place q_issued % 4 is free: that item's softmax was over before the product
                // that qempty has just reported could be issued
                if (elect_one()) {
                    ManyPart &pt = sh.part[q_issued % 4];
                    pt.row0 = it.q.row0, pt.len = it.q.len, pt.n = it.q.n, pt.t0 = it.t0;
                    pt.t1 = it.t1, pt.s = it.s, pt.h = it.h, pt.tiles = it.n;
                    pt.ns = it.ns, pt.lo = it.lo, pt.j0 = j0, pt.j1 = j1;
                    pt.peer = j0 > 0 ? my.share.of(u - j0) : my.share.of(u + it.n - 1) - my.cta;
                }
                __syncwarp();
                if (elect_one()) {
                    const uint32_t bar = smem_u32(&sh.qfull);
                    mbar_expect_tx(bar, 2u * CB * 128u * a.tpt * a.a.group);
                    for (int g = 0; g < 2; ++g)
                        for (int cb = 0; cb < CB; ++cb)
                            tma_load_3d(qbase + g * Cfg::QG + cb * 128 * 128, &qmap, cb * 64, it.h * a.a.group,
                                        it.q.row0 + it.t0 + g * a.tpt, bar);
                }
                __syncwarp();
                ++q_issued;
                next_item(j1);
            }
        } else if (warp == 11) {
            // ---- every V tile passes by here.  Positions that no one wrote, in the box that
            // holds the sequence's end: whatever V has there, 0 * it has to be 0 ----
            bool ok = true;
            uint32_t n = 1;
            while (ok && u < my.u1) {
                const int j1 = part_end();
                for (int j = j0; j < j1; ++j, n += 2) {
                    const uint32_t slot = n % NS;
                    ok = wait(&sh.kvfull[slot], n / NS);
                    if (!ok) break;
                    const int r1 = it.q.len - kv_item_pos<kTileN>(it, j);
                    if (r1 < kTileN && r1 % a.box) {
                        const int rows = a.box - r1 % a.box;
                        for (int i = lane; i < rows * (HD / 8); i += 32) {
                            const int r = r1 + i / (HD / 8), c = i % (HD / 8);
                            const uint32_t at = ring + slot * Cfg::SLOT + (c >> 3) * (kTileN * 128) + r * 128 + ((c & 7) << 4);
                            asm volatile("st.shared.v4.b32 [%0], {%1, %1, %1, %1};" ::"r"(at), "r"(0) : "memory");
                        }
                        fence_proxy_async_smem();
                    }
                    __syncwarp();
                    if (lane == 0) mbar_arrive(smem_u32(&sh.vready[slot]));
                }
                next_item(j1);
            }
        } else {
            // ---- the MMAs: the whole warp in step (its values stay uniform, which the
            // instruction's operands have to be), one lane issues ----
            const uint32_t fmt = a.bf16 ? 1u : 0u;
            const uint32_t id_s = (1u << 4) | (fmt << 7) | (fmt << 10) | ((kTileN >> 3) << 17) | (8u << 24);
            const uint32_t id_o = (1u << 4) | (fmt << 7) | (fmt << 10) | (1u << 16) | ((HD >> 3) << 17) | (8u << 24);
            const uint32_t tu = __shfl_sync(0xFFFFFFFFu, tm, 0);
            const uint64_t qd = sw128_desc(qbase), kd = sw128_desc(ring), vd = v_desc(ring);
            const uint32_t n_tiles = static_cast<uint32_t>(my.u1 - my.u0);
            uint32_t n = 0, q = 0, np = 0;   // ring slots, items and P tiles taken
            bool ok = true;
            auto issue_s = [&](int g, uint32_t slot) {
                const uint64_t qg = qd + ((g * Cfg::QG) >> 4), kg = kd + ((slot * Cfg::SLOT) >> 4);
#pragma unroll
                for (int ks = 0; ks < HD / 16; ++ks) {
                    const uint32_t off = ((ks >> 2) * (128 * 128) + (ks & 3) * 32) >> 4;
                    umma_f16(tu + g * 128, qg + off, kg + off, id_s, ks > 0);
                }
                umma_commit(smem_u32(&sh.sfull[g]));
            };
            // K in ring place n and the V before it are done with once the products issued
            // so far are: one commit for both, after what the softmax waits for
            auto free_pair = [&](uint32_t n) { umma_commit(smem_u32(&sh.kvempty[((n + 1) / 2) % (NS / 2)])); };
            // One loop over all tiles: the next item's first S follows the last P V of the one
            // before it like any other.
            ok = wait(&sh.qfull, 0) && wait(&sh.kvfull[0], 0);
            int left = sh.part[0].j1 - sh.part[0].j0;   // of the item's tiles, this one included
            if (ok) {
                tc_fence_after();
                if (elect_one()) {
                    issue_s(0, 0);
                    issue_s(1, 0);
                    free_pair(0);
                    if (left == 1) umma_commit(smem_u32(&sh.qempty));
                }
                __syncwarp();
            }
            bool fresh = true;   // the item's first tile
            n = 1;
            for (; ok && np < n_tiles; ++np, n += 2) {
                const uint32_t vs = n % NS, vpar = n / NS, kn = (n + 1) % NS, kpar = (n + 1) / NS;
                const bool more = np + 1 < n_tiles, last = left == 1;
                const uint64_t vg = vd + ((vs * Cfg::SLOT) >> 4);
#pragma unroll
                for (int g = 0; g < 2; ++g) {
                    const uint32_t od = tu + 256 + g * HD, pa = tu + g * 128;
                    ok = g == 0 ? wait2(&sh.vready[vs], vpar, &sh.pready[0][0], np) : wait(&sh.pready[1][0], np);
                    if (!ok) break;
                    tc_fence_after();
                    if (elect_one()) {
#pragma unroll
                        for (int ks = 0; ks < kTileN / 32; ++ks)
                            umma_f16_ts(od, pa + ks * 8, vg + ks * (2048 >> 4), id_o, (!fresh || ks > 0) ? 1u : 0u);
                    }
                    __syncwarp();
                    ok = wait(&sh.pready[g][1], np);
                    if (!ok) break;
                    tc_fence_after();
                    if (elect_one()) {
#pragma unroll
                        for (int ks = kTileN / 32; ks < kTileN / 16; ++ks)
                            umma_f16_ts(od, pa + ks * 8, vg + ks * (2048 >> 4), id_o, 1u);
                        if (last) umma_commit(smem_u32(&sh.ofull[g]));
                    }
                    __syncwarp();
                    if (!more) continue;
                    if (g == 0) {
                        ok = wait(&sh.kvfull[kn], kpar);
                        if (ok && last) {   // the next item
                            ok = wait(&sh.qfull, ++q);
                            left = sh.part[q % 4].j1 - sh.part[q % 4].j0 + 1;
                        }
                        if (!ok) break;
                        tc_fence_after();
                    }
                    if (elect_one()) {
                        issue_s(g, kn);
                        if (g == 1) {
                            free_pair(n + 1);
                            if (left == 2) umma_commit(smem_u32(&sh.qempty));   // that was the item's last S
                        }
                    }
                    __syncwarp();
                }
                fresh = last;
                --left;
            }
            // every MMA issued is complete before TMEM is given back
            if (elect_one()) umma_commit(smem_u32(&sh.done));
            __syncwarp();
            mbar_wait_bounded(smem_u32(&sh.done), 0, err, kKvDrain);
        }
    } else {
        // ---- softmax: thread = row ----
        asm volatile("setmaxnreg.inc.sync.aligned.u32 208;");
        const int g = warp >> 2, lr = (warp & 3) * 32 + lane;
        const uint32_t lanes = static_cast<uint32_t>((warp & 3) * 32) << 16;
        const uint32_t ts = tm + g * 128 + lanes, to = tm + 256 + g * HD + lanes;
        const int tok_in = lr / a.a.group, hh = lr - tok_in * a.a.group;
        const float sc = a.a.scale2;
        uint32_t cnt = 0, items = 0, joins = 0;
        int tell = -1;   // the CTA that waits for this one's part
        auto told = [&]() {   // each softmax warp for its rows
            kv_arrive(a.a, tell);
            sh.owed.told[warp] = 1;
            tell = -1;
        };
        bool ok = true;
        auto join = [&]() {   // of the 256 softmax threads; bounded like every wait
            mbar_arrive(smem_u32(&sh.join));
            ok = wait(&sh.join, joins++);
            return ok;
        };
        const uint32_t n_tiles = static_cast<uint32_t>(my.u1 - my.u0);
        while (ok && cnt < n_tiles) {
            ok = wait(&sh.sfull[g], cnt);   // of the item's first tile: its description is there too
            if (!ok) break;
            const ManyPart it = sh.part[items % 4];
            const int j0 = it.j0, j1 = it.j1;
            const int tok = it.t0 + g * a.tpt + tok_in;
            const bool on = tok_in < a.tpt && tok < it.t1;
            const int p0 = it.len - it.n, pos = on ? p0 + tok : -1;
            // the group's first and last position
            const int pmin = p0 + it.t0 + g * a.tpt, pmax = p0 + min(it.t1, it.t0 + (g + 1) * a.tpt) - 1;
            float m = -INFINITY, l = 0.f;
            for (int j = j0; j < j1; ++j) {
                if (j > j0) ok = wait(&sh.sfull[g], cnt);
                if (!ok) break;
                ++cnt;
                tc_fence_after();
                uint32_t s[128];
                tmem_ld32(ts, s);
                tmem_ld32(ts + 32, s + 32);
                tmem_ld32(ts + 64, s + 64);
                tmem_ld32(ts + 96, s + 96);
                tmem_wait_ld(s);
                after_wait(s + 32);
                after_wait(s + 64);
                after_wait(s + 96);
                const int k0 = (j < it.ns ? j : j - it.ns + it.lo) * kTileN;
                if (k0 + kTileN - 1 > pmin) {
                    const int last = pos - k0;   // the last column that the row sees
#pragma unroll
                    for (int c = 0; c < 128; ++c)
                        if (c > last) s[c] = 0xFF800000u;
                }
                if (a.a.window > 0 && k0 <= pmax - a.a.window && k0 + kTileN > a.a.sinks) {
                    const int first = pos - a.a.window + 1 - k0, sinks = a.a.sinks - k0;   // columns below first, past the sinks
#pragma unroll
                    for (int c = 0; c < 128; ++c)
                        if (c < first && c >= sinks) s[c] = 0xFF800000u;
                }
                float mxs[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
                for (int c = 0; c < 128; c += 2)
                    mxs[(c >> 1) & 3] = fmaxf(fmaxf(__uint_as_float(s[c]), __uint_as_float(s[c + 1])), mxs[(c >> 1) & 3]);
                float mx = fmaxf(fmaxf(mxs[0], mxs[1]), fmaxf(mxs[2], mxs[3]));
                mx *= sc;
                // (rows that there are not hold whatever shared memory held: they have no say in
                // when the others rescale, or results would not repeat)
                if (__any_sync(0xFFFFFFFFu, on && mx > m + TOP)) {
                    const float mn = fmaxf(m, mx - UP);
                    const float corr = m == -INFINITY ? 0.f : ex2(m - mn);
                    l *= corr;
                    m = mn;
                    if (j > j0) {
#pragma unroll 1
                        for (int c = 0; c < HD; c += 32) {
                            uint32_t o[32];
                            tmem_ld32(to + c, o);
                            tmem_wait_ld(o);
#pragma unroll
                            for (int i = 0; i < 32; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * corr);
                            tmem_st32(to + c, o);
                        }
                    }
                }
                const float nm = m == -INFINITY ? 0.f : -m;
                const float2 sc2 = make_float2(sc, sc), nm2 = make_float2(nm, nm);
                float2 sum[2] = {make_float2(0.f, 0.f), make_float2(0.f, 0.f)};
                // P in two halves: the product of the first runs while the second is computed.
                // (All exponentials go to the multi-function unit: a polynomial on the FMA pipe for
                // 1 to 4 of 8 measured slower, and so did a first part of three quarters.)
#pragma unroll
                for (int h = 0; h < 2; ++h) {
#pragma unroll
                    for (int c = h * 32; c < h * 32 + 32; ++c) {   // the pairs take the places of scores that are done with
                        float2 x = __ffma2_rn(make_float2(__uint_as_float(s[2 * c]), __uint_as_float(s[2 * c + 1])), sc2, nm2);
                        x.x = ex2(x.x);
                        x.y = ex2(x.y);
                        sum[c & 1] = __fadd2_rn(sum[c & 1], x);
                        if constexpr (BF) {
                            const __nv_bfloat162 w = __floats2bfloat162_rn(x.x, x.y);
                            s[c] = *reinterpret_cast<const uint32_t *>(&w);
                        } else {
                            const __half2 w = __floats2half2_rn(x.x, x.y);
                            s[c] = *reinterpret_cast<const uint32_t *>(&w);
                        }
                    }
                    tmem_st32(ts + h * 32, s + h * 32);
                    tmem_wait_st();
                    tc_fence_before();
                    mbar_arrive(smem_u32(&sh.pready[g][h]));
                }
                l += (sum[0].x + sum[0].y) + (sum[1].x + sum[1].y);
                if (tell >= 0) told();
            }
            if (!ok || !wait(&sh.ofull[g], items)) break;
            const int at_bad = items & 7;
            ++items;
            const bool bad = *reinterpret_cast<volatile int *>(&sh.bad[at_bad]) == static_cast<int>(items);
            tc_fence_after();
            const int row = g * 128 + lr;
            if (j0 > 0) {
                // ---- not the item's beginning: the part goes to the CTA that has it ----
                float *part = a.a.part + static_cast<size_t>(my.cta) * Cfg::PART + row * 4;
#pragma unroll 1
                for (int c = 0; c < HD; c += 32) {
                    uint32_t o[32];
                    tmem_ld32(to + c, o);
                    tmem_wait_ld(o);
                    if (on) {
#pragma unroll
                        for (int i = 0; i < 32; i += 4)
                            __stcg(reinterpret_cast<uint4 *>(part) + ((c + i) / 4) * 256, make_uint4(o[i], o[i + 1], o[i + 2], o[i + 3]));
                    }
                }
                part += 256 * HD - row * 3;
                if (on) {   // rows that there are not stay out of the traffic
                    __stcg(part, m);
                    __stcg(part + 256, bad ? -1.f : l);   // a page outside the pool: a sum that no part has
                }
                // the stores are under way; that they have arrived is told later
                tell = static_cast<int>(it.peer);
            } else {
                // ---- the beginning: the other parts, of the CTAs after this one, are added in
                // order.  They are waited for (as every wait, within a limit): the ranges run
                // against blockIdx, so those CTAs were started before this one. ----
                const unsigned others = it.peer;
                const float *part = a.a.part + static_cast<size_t>(my.cta + 1) * Cfg::PART;
                float M = m, L = l;
                bool odd = bad;
                if (others > 0) {
                    // 8 softmax warps of each of the others
                    if (tid == 0) {
                        if (!kv_await(a.a, my.cta, 8 * others, failed)) {
                            if (!failed()) atomicExch(err, ERR_WAIT_TIMEOUT);
                            *reinterpret_cast<volatile int *>(&sh.fail) = 1;
                        }
                        sh.owed.joined = 1;
                    }
                    if (!join()) break;
                    const unsigned mine_others = on ? others : 0;
#pragma unroll 4
                    for (unsigned c = 0; c < mine_others; ++c) M = fmaxf(M, __ldcg(part + c * Cfg::PART + 256 * HD + row));
                    const float f = m == -INFINITY ? 0.f : ex2(m - M);
                    L = m == -INFINITY ? l : f * l;
#pragma unroll 4
                    for (unsigned c = 0; c < mine_others; ++c) {
                        const float *pp = part + c * Cfg::PART + 256 * HD + row;
                        const float pm = __ldcg(pp), pl = __ldcg(pp + 256);
                        odd = odd | (pl < 0.f);
                        L += pm == -INFINITY ? pl : ex2(pm - M) * pl;
                    }
                    // O in TMEM becomes the item's sum
#pragma unroll 1
                    for (int c = 0; c < HD; c += 64) {
                        uint32_t o[64];
                        float *x = reinterpret_cast<float *>(o);
                        tmem_ld32(to + c, o);
                        tmem_ld32(to + c + 32, o + 32);
                        tmem_wait_ld(o);
                        after_wait(o + 32);
#pragma unroll
                        for (int i = 0; i < 64; ++i) x[i] *= f;
#pragma unroll 1
                        for (unsigned k = 0; k < mine_others; ++k) {
                            const float *pp = part + k * Cfg::PART + row * 4;
                            float4 v[16];
#pragma unroll
                            for (int i = 0; i < 16; ++i) v[i] = __ldcg(reinterpret_cast<const float4 *>(pp) + (c / 4 + i) * 256);
                            const float pm = __ldcg(part + k * Cfg::PART + 256 * HD + row);
                            const float pf = pm == -INFINITY ? 0.f : ex2(pm - M);
#pragma unroll
                            for (int i = 0; i < 16; ++i) {
                                x[4 * i] = fmaf(pf, v[i].x, x[4 * i]);
                                x[4 * i + 1] = fmaf(pf, v[i].y, x[4 * i + 1]);
                                x[4 * i + 2] = fmaf(pf, v[i].z, x[4 * i + 2]);
                                x[4 * i + 3] = fmaf(pf, v[i].w, x[4 * i + 3]);
                            }
                        }
                        tmem_st32(to + c, o);
                        tmem_st32(to + c + 32, o + 32);
                    }
                    tmem_wait_st();
                }
                I *out = static_cast<I *>(const_cast<void *>(a.a.o.p));
                const long long off = on ? (it.row0 + tok) * a.a.o.row + (it.h * a.a.group + hh) * a.a.o.head : -1;
                I *mine = reinterpret_cast<I *>(stage + warp * Cfg::STAGE);   // [32 rows][64], 16-byte pieces swizzled
                const bool bad_page = odd;
                const float inv = L == 0.f ? 0.f : 1.0f / L;
                // Rolled, since this code comes by once an item: unrolled, it would come from
                // beyond the instruction cache every time.
#pragma unroll 1
                for (int c = 0; c < HD; c += 32) {
                    uint32_t o[32];
                    float *x = reinterpret_cast<float *>(o);
                    tmem_ld32(to + c, o);
                    tmem_wait_ld(o);
                    float2 nil = make_float2(0.f, 0.f);   // stays zero where everything is finite
#pragma unroll
                    for (int i = 0; i < 32; i += 2) nil = __ffma2_rn(make_float2(x[i], x[i + 1]), make_float2(0.f, 0.f), nil);
                    // (a sum of numerators that is NaN: a score that the row sees is, and so is the row)
                    odd = odd | (!(nil.x + nil.y == 0.f) && !isnan(L));
#pragma unroll
                    for (int i = 0; i < 32; i += 8) {
                        float y[8];
#pragma unroll
                        for (int e = 0; e < 8; ++e) y[e] = x[i + e] * inv;
                        kv_store8(mine + lane * 64 + ((((c + i) >> 3) ^ lane) & 7) * 8, y);
                    }
                    if (c & 32) {   // 64 dimensions through shared memory, so that 8 lanes write 128 bytes of a row
                        __syncwarp();
#pragma unroll
                        for (int i = 0; i < 8; ++i) {
                            const int r = i * 4 + (lane >> 3), k = lane & 7;
                            const long long ro = __shfl_sync(0xFFFFFFFFu, off, r);
                            const uint4 v = *reinterpret_cast<const uint4 *>(mine + r * 64 + ((k ^ r) & 7) * 8);
                            if (ro >= 0) *reinterpret_cast<uint4 *>(out + ro + c - 32 + k * 8) = v;
                        }
                        __syncwarp();
                    }
                }
                // rows that are not finite: V of a position that a row does not see may have been
                // (0 * NaN), or a page lies outside the pool.  Once more at the end, over their own positions only.
                const unsigned rows = __ballot_sync(0xFFFFFFFFu, odd && on);
                if (rows) {
                    const bool must = __any_sync(0xFFFFFFFFu, bad_page && on);
                    if (lane == 0) sh.again[warp].add(rows, it.t0 + g * a.tpt, it.s, it.h, must);
                }
            }
        }
        if (tell >= 0) told();
        __syncwarp();
        if (sh.again[warp].n > 0) kv_again<HD, I, I, kTileN, true>(a.a, sh.again, 0, a.tpt, a.tpi, a.few_rows, sh.scan);
    }
    // ---- the end: nothing in flight, TMEM given back ----
    tc_fence_before();
    __syncthreads();
    if (sh.fail) {   // a wait ran out: the counters, and the copies still in flight
        if (tid == 0) kv_leave<kTileN, 8>(a.a, a.tpi, a.few_rows, sh.scan, sh.owed);
        if (warp == 9)
            for (uint32_t n = kv_issued > NS ? kv_issued - NS : 0; n < kv_issued; ++n)
                mbar_wait_bounded(smem_u32(&sh.kvfull[n % NS]), (n / NS) & 1u, nullptr, kKvDrain);
        if (warp == 10 && q_issued > 0) mbar_wait_bounded(smem_u32(&sh.qfull), (q_issued - 1) & 1u, nullptr, kKvDrain);
    }
    __syncthreads();
    if (warp == 8) {
        tc_fence_after();
        tmem_dealloc(tm, 512);
    }
}

// ---------------------------------------------------------------------------
// host side
// ---------------------------------------------------------------------------
size_t kv_many_part_bytes() { return sizeof(float) * ManyCfg<128>::PART; }

template <int HD, class I>
static int many_launch(ManyArgs &m, int tc, int sms, cudaStream_t st)
{
    AttnArgs &a = m.a;
    CUtensorMap qm, km, vm;
    int ax[3];
    m.box = kTileN;
    while (a.c.page_size % m.box) m.box >>= 1;   // at least 16: it divides every page
    if (!kv_maps(a.c, HD, tc, m.box, &km, &vm, ax)) return 0;
    a.ax_pos = ax[0], a.ax_head = ax[1], a.ax_page = ax[2];
    // Q: dimension, head, token; boxes of 64 dimensions x G heads x the group's tokens
    const cuuint64_t dims[3] = {static_cast<cuuint64_t>(HD), static_cast<cuuint64_t>(a.nh),
                                static_cast<cuuint64_t>(a.b.n_tokens)};
    const cuuint64_t strides[2] = {static_cast<cuuint64_t>(a.nh > 1 ? a.q.head : HD) * 2,
                                   static_cast<cuuint64_t>(a.b.n_tokens > 1 ? a.q.row : static_cast<long long>(a.nh) * HD) * 2};
    const cuuint32_t box[3] = {64, static_cast<cuuint32_t>(a.group), static_cast<cuuint32_t>(m.tpt)}, estr[3] = {1, 1, 1};
    EncodeTiled enc = encode_tiled();
    if (!enc || enc(&qm, tc == QT_F16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 3,
                    const_cast<void *>(a.q.p), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
                    CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                    CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) != CUDA_SUCCESS) {
        return -1;   // strides that a tensor map cannot have
    }
    auto fn = k_kv_many<HD, I>;
    if (!smem_attr_once(reinterpret_cast<const void *>(fn), ManyCfg<HD>::SMEM)) {
        cudaGetLastError();
        return 0;
    }
    void *args[] = {&qm, &km, &vm, &m};
    return kv_launch(reinterpret_cast<const void *>(fn), dim3(sms < kManyCtas ? sms : kManyCtas), kManyThreads,
                     ManyCfg<HD>::SMEM, args, st);
}

int kv_many_launch(AttnArgs a, int hd, int tc, int few_rows, int sms, cudaStream_t st)
{
    ManyArgs m{a, 128 / a.group, 2 * (128 / a.group), few_rows, 0, tc == QT_BF16};
    if (hd == 128)
        return tc == QT_BF16 ? many_launch<128, __nv_bfloat16>(m, tc, sms, st) : many_launch<128, __half>(m, tc, sms, st);
    return tc == QT_BF16 ? many_launch<64, __nv_bfloat16>(m, tc, sms, st) : many_launch<64, __half>(m, tc, sms, st);
}

}  // namespace tb
