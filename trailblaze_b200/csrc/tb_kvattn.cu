// tb_kvattn.cu — attention of a step's new tokens over the paged cache
// (include/tb_gguf_dequant.h part 4, tb_cuda_kv_attend_dev).
//
// k_kv_few: few query rows per kv head (single tokens, short chunks), bound by
// the cache's bytes.
//
// An item is (sequence, kv head, 8 query rows): row r of a sequence's n * G rows
// (G = query heads per kv head) is new token r / G, head r % G of the group.  Its
// positions come in slices of 16 (16 divides a page), a step is one slice for
// each of the CTA's W warps.  All items' steps (and some more for each item's own
// cost), laid end to end, are cut into equal parts, one per CTA, whatever the
// sequences' lengths: a CTA works through the end of one item, whole items, and the
// beginning of another.  Items that lie
// in one CTA are written out directly, the others' parts go through the workspace to
// the CTA that has the item's beginning, which adds them in CTA order, so results
// repeat bit for bit.
//
// Each warp streams its own slices of K and V through its own ring of TMA copies
// (128-byte swizzle, one mbarrier a stage), with no CTA barrier inside an item.
// The products run on mma.sync with the query rows as N = 8 (a decode step has 4
// to 8 of them; as M they would waste half or more of a 16-row tile and twice the
// registers): S^T[16 positions][8 rows] = K Q^T, O^T[dim][8 rows] += V^T P^T.
// tcgen05's smallest tile is 64 rows of M: at this arithmetic intensity the
// tensor pipe idles either way.
//
// Precision: 16-bit activations over a cache of their type multiply as they are;
// P goes in as a high and a low 16-bit part.  fp16 ends at 2^-24, so over an F16 cache the
// numerators are kept just below the other end of its range, the largest at 2^15: what both
// parts lose of one lies 2^-40 below the largest (at 1, 2^-25 below it: where one position
// outweighs the rest by 2^25, the rest would vanish).  fp32 activations are split into
// parts of the cache's type (3 bf16, or 2 fp16 of a row scaled by a power of two
// so that its largest element is near 2^13); an fp32 cache is split into two
// tf32 parts, of which the low-low product is dropped (2^-22).  Scores, softmax and
// sums are fp32.
//
// Measured (8 kv heads of 128, 4 query heads each): 64 sequences of up to 16384 bf16
// positions, 2.07 GB, in 307 to 338 us by the GPU, 6.1 to 6.7 TB/s, where a copy reaches
// 6.5; one sequence of 4096 fp32 positions, 33.6 MB, in 19 us against 5 us of bytes:
// launch, scan, the first page, Q and the joining of 16 parts stand one behind the other
// there.
#include "../../include/tb_gguf_dequant.h"
#include "tb_kvattn.cuh"

namespace tb {

// ---- the layout of an item's positions ----
static constexpr int kSlice = 16;

// The slices that any row of a sequence sees: [0, ns) and [lo, lo + n - ns).
struct KvSlices {
    int ns, lo, n;
};
__device__ __forceinline__ KvSlices kv_slices(const KvSeq &q, int window, int sinks)
{
    const KvSpan sp = kv_span(q.len - q.n, window, sinks);   // of the first row, which sees furthest back
    const int all = (q.len + kSlice - 1) / kSlice;
    KvSlices s{0, 0, all};
    if (sinks < sp.lo) {
        s.ns = (sinks + kSlice - 1) / kSlice;
        s.lo = sp.lo / kSlice > s.ns ? sp.lo / kSlice : s.ns;
        s.n = s.ns + all - s.lo;
    }
    return s;
}

struct FewShared {
    float m[8][8], l[8][8];   // [warp][row]
    unsigned long long scan[8], items[8], at;
    int seq, fail, bad[8];
};

template <int HD, int TI, int TC>
struct FewCfg {
    static constexpr int ES = TC == QT_F32 ? 4 : 2;
    static constexpr int SB = kSlice * HD * ES;                 // bytes of a slice of K or of V
    // 8 warps on one CTA an SM for the slices that take the most arithmetic a byte's
    // copy (fp32, 128 dimensions), else two CTAs of 4: one streams while the other
    // joins its warps.  24 KB a warp in flight either way.
    static constexpr int W = SB >= 8192 ? 8 : 4;                // warps
    static constexpr int CTAS = SB >= 8192 ? 1 : 2;             // per SM
    static constexpr int NST = SB >= 8192 ? 3 : SB >= 4096 ? 6 : 12;
    static constexpr int MIN = SB >= 8192 ? 2 : 4;              // steps of a CTA, at least
    // An item's own cost (Q, the joining of the warps, output: some 3 us), in steps at the
    // rate of a CTA's share of the bandwidth: it counts in the cutting, else the CTAs that
    // get many short sequences finish last (24 sequences of up to 1733 positions, 16 heads
    // of 64: 50 us without)
    static constexpr int COST = 65536 / (W * 2 * SB) > 0 ? 65536 / (W * 2 * SB) : 1;
    static constexpr int NQ = TC == QT_F32 ? 2 : TI == TC ? 1 : TC == QT_BF16 ? 3 : 2;
    static constexpr int NP = TC == QT_BF16 && TI == QT_F32 ? 3 : 2;
    static constexpr int MERGE = W * 8 * HD * 4;
    // Rings, merge buffer, barriers, FewShared.  Nothing static and no slack for
    // alignment, so that two CTAs fit an SM: the block's window begins on a 1 KB
    // boundary, which the kernel checks.
    static constexpr int SMEM = W * NST * SB + MERGE + W * NST * 8 + static_cast<int>(sizeof(FewShared));
};
// floats of one partial result: 8 rows of O, then m and l of each
__host__ __device__ constexpr int few_part(int hd) { return 8 * hd + 16; }

// True for a sequence of this launch.
__device__ __forceinline__ bool few_seq(const AttnArgs &a, const KvSeq &q)
{
    return q.n > 0 && static_cast<long long>(q.n) * a.group <= a.many_rows;
}

// A place in the sequence of all items' steps.
struct KvCur {
    int s, h, rt, step;     // sequence, kv head, row tile, step
    KvSeq q;
    KvSlices sl;
    int tiles, steps;       // row tiles per head, steps per item
};

template <int W>
__device__ __forceinline__ void kv_cur_seq(const AttnArgs &a, KvCur &c)
{
    // sequences that cannot be are skipped here; the scan has reported them
    while (c.s < a.b.n_seqs && (!kv_seq(a.b, a.c, c.s, c.q, nullptr) || !few_seq(a, c.q))) ++c.s;
    if (c.s >= a.b.n_seqs) return;
    c.sl = kv_slices(c.q, a.window, a.sinks);
    c.tiles = (c.q.n * a.group + 7) >> 3;
    c.steps = (c.sl.n + W - 1) / W;
}

template <int W, int COST>
__device__ __forceinline__ unsigned long long kv_seq_steps(const AttnArgs &a, int s, bool &bad, unsigned long long *items)
{
    KvSeq q;
    if (!kv_seq(a.b, a.c, s, q, nullptr)) {
        bad = true;
        return 0;
    }
    if (!few_seq(a, q)) return 0;
    const KvSlices sl = kv_slices(q, a.window, a.sinks);
    const unsigned long long tiles = (static_cast<unsigned long long>(q.n) * a.group + 7) >> 3;
    if (items) *items += tiles * a.c.n_kv_heads;
    return tiles * a.c.n_kv_heads * static_cast<unsigned>((sl.n + W - 1) / W + COST);
}

template <int HD, int TI, int TC>
__global__ void __launch_bounds__(FewCfg<HD, TI, TC>::W * 32, FewCfg<HD, TI, TC>::CTAS)
    k_kv_few(const __grid_constant__ CUtensorMap kmap, const __grid_constant__ CUtensorMap vmap, const AttnArgs a)
{
    using Cfg = FewCfg<HD, TI, TC>;
    using I = typename KvType<TI>::E;
    using E = typename KvType<TC>::E;
    constexpr int W = Cfg::W, T = W * 32, NST = Cfg::NST, NQ = Cfg::NQ, NP = Cfg::NP, ES = Cfg::ES;
    constexpr bool X32 = TC == QT_F32;
    constexpr bool FINE = TI == QT_F32;          // fp32 results
    constexpr int NC = FINE ? 5 : 2;             // accumulators of a score: 4 and the small products', or 2
    // Numerators are 2^(score - m): m follows the running maximum, moved when a score passes
    // it by 2^TOP, to 2^UP below the largest score then.
    constexpr float TOP = TC == QT_F16 ? 15.f : 8.f, UP = TC == QT_F16 ? 15.f : 0.f;
    constexpr int KS = X32 ? HD / 8 : HD / 16;   // steps of the product over the head's dimensions
    constexpr int CB = HD * ES / 128;            // 128-byte columns of a row
    constexpr uint32_t kCol = kSlice * 128;
    extern __shared__ __align__(1024) uint8_t sm[];
    float *merge = reinterpret_cast<float *>(sm + W * NST * Cfg::SB);   // [W][8][HD]
    uint64_t *full = reinterpret_cast<uint64_t *>(merge + Cfg::MERGE / 4);
    FewShared &sh = *reinterpret_cast<FewShared *>(full + W * NST);
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, t = lane & 3;

    if (smem_u32(sm) & 1023u) {   // the swizzle of the copies goes by address bits
        if (tid == 0) atomicExch(a.err, ERR_RUNTIME);
        return;
    }
    if (tid == 0) {
        for (int i = 0; i < W * NST; ++i) mbar_init(smem_u32(full + i), 1);
        fence_mbar_init();
        sh.fail = 0;
        sh.seq = a.b.n_seqs;
    }
    if (tid < 2) prefetch_map(tid ? &vmap : &kmap);
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    asm volatile("griddepcontrol.wait;" ::: "memory");
    // ---- this CTA's share of all steps: a scan over the sequences ----
    const int per = (a.b.n_seqs + T - 1) / T, sq0 = tid * per, sq1 = min(a.b.n_seqs, sq0 + per);
    unsigned long long mine = 0, items = 0;
    bool bad_seq = false;
    for (int s = sq0; s < sq1; ++s) mine += kv_seq_steps<W, Cfg::COST>(a, s, bad_seq, &items);
    if (__syncthreads_or(bad_seq) && blockIdx.x == 0) kv_zero_bad<HD, I>(a);
    unsigned long long incl = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const unsigned long long x = __shfl_up_sync(0xFFFFFFFFu, incl, o);
        if (lane >= o) incl += x;
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) items += __shfl_xor_sync(0xFFFFFFFFu, items, o);
    if (lane == 31) sh.scan[warp] = incl, sh.items[warp] = items;
    __syncthreads();
    unsigned long long before = incl - mine, total = 0, all_items = 0;
#pragma unroll
    for (int w = 0; w < W; ++w) {
        all_items += sh.items[w];
        before += w < warp ? sh.scan[w] : 0;
        total += sh.scan[w];
    }
    // A CTA for every item, or more, with at least MIN steps each (128 KB of the cache):
    // finer cuts gain less than the joining of their parts costs.
    if (total == 0) return;
    const unsigned long long most = min(max(all_items, (total + Cfg::MIN - 1) / Cfg::MIN), static_cast<unsigned long long>(gridDim.x));
    const unsigned long long longest = kv_div(total + most - 1, most);
    const unsigned G = static_cast<unsigned>(kv_div(total + longest - 1, longest));
    if (blockIdx.x >= G) return;
    const unsigned cta = G - 1 - blockIdx.x;   // of the steps, against blockIdx: see the joining of parts
    const KvShare share(total, G);
    const unsigned long long u0 = share.start(cta), u1 = share.start(cta + 1);
    if (before <= u0 && u0 < before + mine) {
        unsigned long long at = before;
        for (int s = sq0; s < sq1; ++s) {
            const unsigned long long n = kv_seq_steps<W, Cfg::COST>(a, s, bad_seq, nullptr);
            if (u0 < at + n) {
                sh.seq = s;
                sh.at = u0 - at;
                break;
            }
            at += n;
        }
    }
    __syncthreads();

    KvCur cu{};
    cu.s = sh.seq;
    kv_cur_seq<W>(a, cu);
    {
        const unsigned long long r = sh.at, item = kv_div(r, cu.steps + Cfg::COST), head = kv_div(item, cu.tiles);
        cu.step = static_cast<int>(r - item * (cu.steps + Cfg::COST)) - Cfg::COST;
        cu.rt = static_cast<int>(item - head * cu.tiles);
        cu.h = static_cast<int>(head);
    }
    auto advance_item = [&](KvCur &c) {
        c.step = -Cfg::COST;
        if (++c.rt < c.tiles) return;
        c.rt = 0;
        if (++c.h < a.c.n_kv_heads) return;
        c.h = 0;
        ++c.s;
        kv_cur_seq<W>(a, c);
    };

    // ---- the warp's ring ----
    const uint32_t ring = smem_u32(sm) + warp * NST * Cfg::SB;
    const uint32_t bars = smem_u32(full) + warp * NST * 8;
    KvCur ic = cu;                              // the next step to be requested
    unsigned long long iu = u0;
    uint32_t issued = 0, taken = 0;             // tiles (K and V of a slice in turn) requested / consumed
    uint32_t hidden = 0;                        // bit st: stage st's page is outside the pool
    int pg = -1, pg_s = -1, pg_base = 0;        // lane l: the page of the warp's slice in step pg_base + l
    int cy = 0, cz = 0, cw = 0;                 // the last slice's coordinates
    bool v_due = false, cbad = false, ok = true;
    auto request = [&](const CUtensorMap *map) {
        const uint32_t st = issued % NST, bar = bars + st * 8, dst = ring + st * Cfg::SB;
        hidden = cbad ? hidden | (1u << st) : hidden & ~(1u << st);
        if (lane == 0) {
            if (cbad) {
                mbar_arrive(bar);
            } else {
                mbar_expect_tx(bar, Cfg::SB);
#pragma unroll
                for (int cb = 0; cb < CB; ++cb) tma_load_4d(dst + cb * kCol, map, cb * (128 / ES), cy, cz, cw, bar);
            }
        }
        ++issued;
    };
    auto issue_step = [&]() {   // K of the warp's slice of step iu, if it has one
        const int sl = ic.step * W + warp;
        if (ic.step >= 0 && sl < ic.sl.n) {
            if (ic.s != pg_s || ic.step >= pg_base + 32 || ic.step < pg_base) {
                pg_s = ic.s, pg_base = ic.step;
                const int my = (ic.step + lane) * W + warp;
                pg = -1;
                if (my < ic.sl.n) {
                    const int j = (my < ic.sl.ns ? my : my - ic.sl.ns + ic.sl.lo) * kSlice;
                    pg = a.b.pages[static_cast<long long>(ic.s) * a.b.pages_stride + fdiv(static_cast<uint32_t>(j), a.c.page_div)];
                }
            }
            const int page = __shfl_sync(0xFFFFFFFFu, pg, ic.step - pg_base);
            const int j = (sl < ic.sl.ns ? sl : sl - ic.sl.ns + ic.sl.lo) * kSlice;
            const int pos = j - static_cast<int>(fdiv(static_cast<uint32_t>(j), a.c.page_div)) * a.c.page_size;
            cbad = page < 0 || page >= a.c.n_pages;
            if (cbad && lane == 0) atomicExch(a.err, ERR_RUNTIME);
            cy = a.ax_pos == 0 ? pos : a.ax_head == 0 ? ic.h : page;
            cz = a.ax_pos == 1 ? pos : a.ax_head == 1 ? ic.h : page;
            cw = a.ax_pos == 2 ? pos : a.ax_head == 2 ? ic.h : page;
            request(&kmap);
            v_due = true;
        }
        ++iu;
        if (++ic.step == ic.steps && iu < u1) {
            advance_item(ic);
            // its Q towards L1 while this item still runs: a row's bytes by 128 a lane
            constexpr int LINES = HD * static_cast<int>(sizeof(I)) / 128;
            const int r = ic.rt * 8 + lane / LINES;
            if (lane < 8 * LINES && r < ic.q.n * a.group) {
                const int tok = r / a.group;
                const I *qp = static_cast<const I *>(a.q.p) + (ic.q.row0 + tok) * a.q.row +
                              (ic.h * a.group + (r - tok * a.group)) * a.q.head + (lane % LINES) * (128 / sizeof(I));
                asm volatile("prefetch.global.L1 [%0];" ::"l"(qp));
            }
        }
    };
    auto refill = [&]() {
        while (ok && issued - taken < NST) {
            if (v_due) {
                request(&vmap);
                v_due = false;
            } else if (iu < u1) {
                issue_step();
            } else {
                break;
            }
        }
    };
    int tell = -1;   // the CTA that waits for this one's part
    auto told = [&]() {
        kv_arrive(a, tell);
        tell = -1;
    };
    const uint32_t krow = (lane & 7) + ((lane >> 3) & 1) * 8, kchunk = lane >> 4;   // ldmatrix rows of K
    const uint32_t vrow = (lane & 7) + (lane >> 4) * 8, vchunk = (lane >> 3) & 1;   // and of V, transposed
    for (unsigned long long u = u0; u < u1;) {
        // ---- one item, or this CTA's part of it ----
        const int step0 = max(cu.step, 0);
        const unsigned long long left = u1 - u;
        const int end = left < static_cast<unsigned>(cu.steps - cu.step) ? cu.step + static_cast<int>(left) : cu.steps;
        const int nstep = end - step0;
        const unsigned long long first = u - cu.step;   // the unit of the item's step 0 (cu.step may be negative)
        if (nstep <= 0) {   // of this item the CTA has only units that stand for its cost
            u += end - cu.step;
            cu.step = end;
            if (u < u1 && cu.step == cu.steps) advance_item(cu);
            continue;
        }
        const bool from_start = cu.step <= 0, to_end = end == cu.steps;
        const int R = cu.q.n * a.group, p0 = cu.q.len - cu.q.n, r0 = cu.rt * 8;
        // row g of Q as the B operand; rows past the last are zero.  It is requested before
        // the ring's copies, behind which it would wait.
        uint32_t qf[NQ][KS][2];
        float rscale = a.scale2;
        {
            constexpr int QE = X32 ? 2 : 4;   // elements of a step
            const int r = r0 + g, tok = r / a.group;
            const bool on = r < R;
            const I *qp = static_cast<const I *>(a.q.p) + (cu.q.row0 + (on ? tok : 0)) * a.q.row +
                          (cu.h * a.group + (on ? r - tok * a.group : 0)) * a.q.head;
            if constexpr (NQ == 1) {
#pragma unroll
                for (int ks = 0; ks < KS; ++ks)
#pragma unroll
                    for (int e = 0; e < 2; ++e)
                        qf[0][ks][e] = on ? *reinterpret_cast<const uint32_t *>(qp + ks * 16 + 2 * t + 8 * e) : 0u;
                refill();
            } else {
                I x[KS][QE];
#pragma unroll
                for (int ks = 0; ks < KS; ++ks)
#pragma unroll
                    for (int e = 0; e < QE; ++e)
                        x[ks][e] = qp[X32 ? ks * 8 + t + 4 * e : ks * 16 + 2 * t + 8 * (e >> 1) + (e & 1)];
                refill();
                float y[KS][QE], big = 0.f;
#pragma unroll
                for (int ks = 0; ks < KS; ++ks)
#pragma unroll
                    for (int e = 0; e < QE; ++e) {
                        y[ks][e] = on ? kv_f(x[ks][e]) : 0.f;
                        big = fmaxf(big, fabsf(y[ks][e]));
                    }
                if constexpr (X32) {
#pragma unroll
                    for (int ks = 0; ks < KS; ++ks)
#pragma unroll
                        for (int e = 0; e < 2; ++e) split_tf32(__float_as_uint(y[ks][e]), qf[0][ks][e], qf[1][ks][e]);
                } else {
                    if constexpr (TC == QT_F16) {   // the row times 2^k, its largest element near 2^13
                        big = fmaxf(big, __shfl_xor_sync(0xFFFFFFFFu, big, 1));
                        big = fmaxf(big, __shfl_xor_sync(0xFFFFFFFFu, big, 2));
                        int k = 0;
                        if (big > 0.f && big < INFINITY) k = 13 - ilogbf(big);
                        k = max(-100, min(100, k));
                        const float up = ldexpf(1.f, k);
                        rscale = ldexpf(a.scale2, -k);
#pragma unroll
                        for (int ks = 0; ks < KS; ++ks)
#pragma unroll
                            for (int e = 0; e < QE; ++e) y[ks][e] *= up;
                    }
#pragma unroll
                    for (int ks = 0; ks < KS; ++ks)
#pragma unroll
                        for (int e = 0; e < 2; ++e)
#pragma unroll
                            for (int n = 0; n < NQ; ++n) qf[n][ks][e] = pack16<TC>(y[ks][2 * e], y[ks][2 * e + 1]);
                }
            }
        }
        if (tell >= 0) told();
        // columns 2 t and 2 t + 1 of S^T and O^T: their positions (-1: no row) and scales
        int pos[2];
        float rs[2];
#pragma unroll
        for (int e = 0; e < 2; ++e) {
            const int r = r0 + 2 * t + e;
            pos[e] = r < R ? p0 + r / a.group : -1;
            rs[e] = __shfl_sync(0xFFFFFFFFu, rscale, (2 * t + e) * 4);
        }
        const int pmin = p0 + r0 / a.group, pmax = p0 + (min(r0 + 8, R) - 1) / a.group;
        float O[HD / 16][4], m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f};
#pragma unroll
        for (int i = 0; i < HD / 16; ++i)
#pragma unroll
            for (int e = 0; e < 4; ++e) O[i][e] = 0.f;

        for (int k = 0; k < nstep; ++k) {
            const int sl = (step0 + k) * W + warp;
            if (sl < cu.sl.n && ok) {
                uint32_t st = taken % NST;
                const int j0 = (sl < cu.sl.ns ? sl : sl - cu.sl.ns + cu.sl.lo) * kSlice;
                ok = mbar_wait_bounded(bars + st * 8, (taken / NST) & 1u, a.err, a.wait_limit);
                ok = __all_sync(0xFFFFFFFFu, ok);
                if (!ok) {
                    sh.fail = 1;
                    break;
                }
                const uint32_t kb = shared_after(ring + st * Cfg::SB);
                const bool bad = (hidden >> st) & 1u;
                // ---- S^T = K Q^T; the tensor core truncates what it adds to an accumulator, so
                // fp32 results come from short chains that are added in fp32, the small
                // products by themselves ----
                float c[NC][4];
#pragma unroll
                for (int i = 0; i < NC; ++i)
#pragma unroll
                    for (int e = 0; e < 4; ++e) c[i][e] = 0.f;
#pragma unroll
                for (int ks = 0; ks < KS; ++ks) {
                    const uint32_t ch = 2 * ks + kchunk;
                    uint32_t x[4];
                    ldsm4(kb + (ch >> 3) * kCol + krow * 128 + (((ch & 7) ^ (krow & 7)) << 4), x);
                    if constexpr (X32) {
                        uint32_t hi[4], lo[4];
#pragma unroll
                        for (int e = 0; e < 4; ++e) split_tf32(x[e], hi[e], lo[e]);
                        mma_tf32(c[NC - 1], lo, qf[0][ks][0], qf[0][ks][1]);
                        mma_tf32(c[NC - 1], hi, qf[1][ks][0], qf[1][ks][1]);
                        mma_tf32(c[FINE ? ks & 3 : ks & 1], hi, qf[0][ks][0], qf[0][ks][1]);
                    } else {
#pragma unroll
                        for (int n = NQ - 1; n >= 0; --n)
                            mma16<TC>(c[n > 0 ? NC - 1 : FINE ? ks & 3 : ks & 1], x, qf[n][ks][0], qf[n][ks][1]);
                    }
                }
#pragma unroll
                for (int i = 0; i < NC; ++i) pin(c[i]);
                __syncwarp();   // every lane has read K
                ++taken;
                refill();
                float x[4];   // (position g, row 2 t), (g, 2 t + 1), (g + 8, 2 t), (g + 8, 2 t + 1)
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    float sum = c[NC - 1][e];   // the small products, or the second chain
                    if constexpr (FINE) sum = ((c[0][e] + c[1][e]) + (c[2][e] + c[3][e])) + sum;
                    else sum += c[0][e];
                    x[e] = sum * rs[e & 1];
                }
                if (bad || j0 + kSlice - 1 > pmin ||
                    (a.window > 0 && j0 <= pmax - a.window && j0 + kSlice > a.sinks)) {
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const int j = j0 + g + 8 * (e >> 1), p = pos[e & 1];
                        const bool see = !bad && j <= p && (a.window == 0 || p - j < a.window || j < a.sinks);
                        x[e] = see ? x[e] : -INFINITY;
                    }
                }
                // ---- m: see TOP and UP ----
                if (__any_sync(0xFFFFFFFFu, fmaxf(x[0], x[2]) > m[0] + TOP || fmaxf(x[1], x[3]) > m[1] + TOP)) {
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        float mx = fmaxf(x[e], x[e + 2]);
#pragma unroll
                        for (int o = 4; o < 32; o <<= 1) mx = fmaxf(mx, __shfl_xor_sync(0xFFFFFFFFu, mx, o));
                        mx = fmaxf(mx - UP, m[e]);
                        const float corr = m[e] == -INFINITY ? 0.f : ex2(m[e] - mx);
                        m[e] = mx;
                        l[e] *= corr;
#pragma unroll
                        for (int i = 0; i < HD / 16; ++i) O[i][e] *= corr, O[i][e + 2] *= corr;
                    }
                }
#pragma unroll
                for (int e = 0; e < 4; ++e) x[e] = ex2(x[e] - (m[e & 1] == -INFINITY ? 0.f : m[e & 1]));
                l[0] += x[0] + x[2];
                l[1] += x[1] + x[3];
                // ---- O^T += V^T P^T ----
                st = taken % NST;
                ok = mbar_wait_bounded(bars + st * 8, (taken / NST) & 1u, a.err, a.wait_limit);
                ok = __all_sync(0xFFFFFFFFu, ok);
                if (!ok) {
                    sh.fail = 1;
                    break;
                }
                uint32_t vb = ring + st * Cfg::SB;
                if (bad || j0 + kSlice > cu.q.len) {
                    // positions that no one wrote (all of them where the page is none): whatever
                    // lies there, 0 * it has to be 0
                    const int r1 = bad ? 0 : cu.q.len - j0;
                    for (int i = lane; i < (kSlice - r1) * (HD * ES / 16); i += 32) {
                        const int r = r1 + i / (HD * ES / 16), c = i % (HD * ES / 16);
                        const uint32_t at = vb + (c >> 3) * kCol + r * 128 + ((c & 7) << 4);
                        asm volatile("st.shared.v4.b32 [%0], {%1, %1, %1, %1};" ::"r"(at), "r"(0) : "memory");
                    }
                    fence_proxy_async_smem();   // before the stage's next copy
                    __syncwarp();
                }
                vb = shared_after(vb);
                if constexpr (X32) {
                    uint32_t ph[2][2], pl[2][2];   // [8 positions][2 t and 2 t + 1 of them, row g]
#pragma unroll
                    for (int kb8 = 0; kb8 < 2; ++kb8)
#pragma unroll
                        for (int e = 0; e < 2; ++e) {
                            const int from = (2 * t + e) * 4 + (g >> 1);
                            const float y0 = __shfl_sync(0xFFFFFFFFu, x[2 * kb8], from);
                            const float y1 = __shfl_sync(0xFFFFFFFFu, x[2 * kb8 + 1], from);
                            split_tf32(__float_as_uint((g & 1) ? y1 : y0), ph[kb8][e], pl[kb8][e]);
                        }
#pragma unroll
                    for (int kb8 = 0; kb8 < 2; ++kb8)
#pragma unroll
                        for (int jb = 0; jb < HD / 64; ++jb) {
                            uint4 v[2][2];   // [column 2 jb, 2 jb + 1][position 2 t, 2 t + 1]: 4 dimensions each
#pragma unroll
                            for (int cc = 0; cc < 2; ++cc)
#pragma unroll
                                for (int e = 0; e < 2; ++e) {
                                    const uint32_t r = kb8 * 8 + 2 * t + e;
                                    v[cc][e] = lds_u128(vb + (2 * jb + cc) * kCol + r * 128 + ((g ^ (r & 7)) << 4));
                                }
#pragma unroll
                            for (int d = 0; d < 4; ++d) {
                                uint32_t hi[4], lo[4];
#pragma unroll
                                for (int e = 0; e < 4; ++e) {
                                    const uint4 &w = v[e & 1][e >> 1];
                                    split_tf32(d == 0 ? w.x : d == 1 ? w.y : d == 2 ? w.z : w.w, hi[e], lo[e]);
                                }
                                float o[4] = {0.f, 0.f, 0.f, 0.f};   // added in fp32: see S^T
                                mma_tf32(o, lo, ph[kb8][0], ph[kb8][1]);
                                mma_tf32(o, hi, pl[kb8][0], pl[kb8][1]);
                                mma_tf32(o, hi, ph[kb8][0], ph[kb8][1]);
#pragma unroll
                                for (int e = 0; e < 4; ++e) O[jb * 4 + d][e] += o[e];
                            }
                        }
                } else {
                    uint32_t pb[NP][2];
#pragma unroll
                    for (int n = 0; n < NP; ++n)
#pragma unroll
                        for (int e = 0; e < 2; ++e) pb[n][e] = mat_t(pack16<TC>(x[2 * e], x[2 * e + 1]));
#pragma unroll
                    for (int i = 0; i < HD / 16; ++i) {
                        const uint32_t ch = 2 * i + vchunk;
                        uint32_t v[4];
                        ldsm4t(vb + (ch >> 3) * kCol + vrow * 128 + (((ch & 7) ^ (vrow & 7)) << 4), v);
                        if constexpr (FINE) {
                            float o[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                            for (int n = NP - 1; n >= 0; --n) mma16<TC>(o, v, pb[n][0], pb[n][1]);
#pragma unroll
                            for (int e = 0; e < 4; ++e) O[i][e] += o[e];
                        } else {
#pragma unroll
                            for (int n = NP - 1; n >= 0; --n) mma16<TC>(O[i], v, pb[n][0], pb[n][1]);
                        }
                    }
                }
#pragma unroll
                for (int i = 0; i < HD / 16; ++i) pin(O[i]);
                __syncwarp();   // every lane has read V
                ++taken;
                refill();
            }
        }
        // ---- the warps' parts of the item, added in warp order ----
#pragma unroll
        for (int e = 0; e < 2; ++e) {
#pragma unroll
            for (int o = 4; o < 32; o <<= 1) l[e] += __shfl_xor_sync(0xFFFFFFFFu, l[e], o);
            if (g == 0) sh.m[warp][2 * t + e] = m[e], sh.l[warp][2 * t + e] = l[e];
#pragma unroll
            for (int i = 0; i < HD / 16; ++i)
#pragma unroll
                for (int k = 0; k < 2; ++k) {
                    const int d = X32 ? (i >> 2) * 64 + k * 32 + 4 * g + (i & 3) : i * 16 + k * 8 + g;
                    merge[(warp * 8 + 2 * t + e) * HD + d] = O[i][e + 2 * k];
                }
        }
        if (tid < 8) sh.bad[tid] = 0;
        __syncthreads();
        const int rows = min(8, R - r0);
        constexpr int PER = 8 * HD / T;                  // consecutive dimensions of one row a thread
        constexpr int RT = HD / PER;                     // threads a row
        const int mr = tid / RT, md = (tid % RT) * PER;  // the thread's row and first dimension
        float M = -INFINITY, L = 0.f, acc[PER];
#pragma unroll
        for (int d = 0; d < PER; ++d) acc[d] = 0.f;
#pragma unroll
        for (int w = 0; w < W; ++w) M = fmaxf(M, sh.m[w][mr]);
#pragma unroll
        for (int w = 0; w < W; ++w) {
            const float f = sh.m[w][mr] == -INFINITY ? 0.f : ex2(sh.m[w][mr] - M);
            // a warp that saw nothing of the row has l = 0, unless what it saw was NaN
            L += sh.m[w][mr] == -INFINITY ? sh.l[w][mr] : f * sh.l[w][mr];
#pragma unroll
            for (int d = 0; d < PER; ++d) acc[d] = fmaf(f, merge[(w * 8 + mr) * HD + md + d], acc[d]);
        }
        bool odd = !isfinite(L) || M == INFINITY;
#pragma unroll
        for (int d = 0; d < PER; ++d) odd = odd || !isfinite(acc[d]);
        if (__syncthreads_or(odd && mr < rows && !sh.fail)) {
            // a row that is not finite: V of a position that this row does not see may have
            // been (0 * NaN).  Such rows once more, over their own positions only.
            if (odd) sh.bad[mr] = 1;
            __syncthreads();
            const int ja = step0 * W, jb = min(cu.sl.n, (step0 + nstep) * W);   // the part's slices
            for (int r = warp; r < rows; r += W) {
                if (!sh.bad[r]) continue;
                const int tok = (r0 + r) / a.group, hh = (r0 + r) - tok * a.group;
                const I *qp = static_cast<const I *>(a.q.p) + (cu.q.row0 + tok) * a.q.row + (cu.h * a.group + hh) * a.q.head;
                // its slices before and after the gap between the first tokens and the window
                const int b0 = min(ja, cu.sl.ns), b1 = min(jb, cu.sl.ns);
                const int c0 = max(ja, cu.sl.ns) - cu.sl.ns + cu.sl.lo, c1 = max(jb, cu.sl.ns) - cu.sl.ns + cu.sl.lo;
                float m = -INFINITY, l = 0.f, o[8];
#pragma unroll
                for (int d = 0; d < 8; ++d) o[d] = 0.f;
#pragma unroll 1
                for (int part = 0; part < 2; ++part) {
                    const I *const q1[1] = {qp};
                    const int i1[1] = {p0 + tok};
                    float xm[1], xl[1], x[1][8];
                    kv_rows_attend<HD, I, E, 1, 4>(a, q1, cu.s, cu.h, i1, (part ? c0 : b0) * kSlice,
                                                part ? min(c1 * kSlice, cu.q.len) : b1 * kSlice, xm, xl, x);
                    const float mm = fmaxf(m, xm[0]);
                    const float f0 = m == -INFINITY ? 0.f : ex2(m - mm), f1 = xm[0] == -INFINITY ? 0.f : ex2(xm[0] - mm);
                    l = (m == -INFINITY ? l : l * f0) + (xm[0] == -INFINITY ? xl[0] : xl[0] * f1);
#pragma unroll
                    for (int d = 0; d < 8; ++d) o[d] = o[d] * f0 + x[0][d] * f1;
                    m = mm;
                }
                if (lane < HD / 8) {
#pragma unroll
                    for (int d = 0; d < 8; ++d) merge[r * HD + lane * 8 + d] = o[d];
                }
                if (lane == 0) sh.m[0][r] = m, sh.l[0][r] = l;
            }
            __syncthreads();
            if (mr < rows && sh.bad[mr]) {
                M = sh.m[0][mr];
                L = sh.l[0][mr];
#pragma unroll
                for (int d = 0; d < PER; ++d) acc[d] = merge[mr * HD + md + d];
            }
        }
        auto write_out = [&]() {
            if (mr >= rows) return;
            const int tok = (r0 + mr) / a.group, hh = (r0 + mr) - tok * a.group;
            I *op = static_cast<I *>(const_cast<void *>(a.o.p)) + (cu.q.row0 + tok) * a.o.row +
                    (cu.h * a.group + hh) * a.o.head + md;
            const float inv = L == 0.f ? 0.f : 1.0f / L;
#pragma unroll
            for (int d = 0; d < PER; ++d) acc[d] = L == 0.f ? 0.f : acc[d] * inv;
            if constexpr (PER == 8) {
                kv_store8(op, acc);
            } else {
#pragma unroll
                for (int d = 0; d < PER; ++d) kv_store1(op + d, acc[d]);
            }
        };
        constexpr int P = few_part(HD);
        if (!from_start) {
            // ---- not the item's beginning: the part goes to the CTA that has it ----
            float *mp = a.part + static_cast<size_t>(cta) * P;
            if (mr < rows) {
#pragma unroll
                for (int d = 0; d < PER; d += 4)
                    __stcg(reinterpret_cast<float4 *>(mp + mr * HD + md + d),
                           make_float4(acc[d], acc[d + 1], acc[d + 2], acc[d + 3]));
                if (md == 0) __stcg(mp + 8 * HD + mr, M), __stcg(mp + 8 * HD + 8 + mr, L);
            }
            // the stores are under way; that they have arrived is told later
            tell = static_cast<int>(share.of(first));
        } else {
            if (!to_end) {
                // ---- the beginning: the other parts, of the CTAs after this one, in order.  They
                // are waited for (as every wait, within a limit): the ranges run against blockIdx,
                // so those CTAs were started before this one. ----
                const unsigned others = share.of(first + cu.steps - 1) - cta;
                const float *part = a.part + static_cast<size_t>(cta + 1) * P;
                if (tid == 0 && !kv_await(a, cta, W * others, [] { return false; })) {
                    atomicExch(a.err, ERR_WAIT_TIMEOUT);
                    sh.fail = 1;
                }
                __syncthreads();
                if (mr < rows) {
                    constexpr int AHEAD = 64 / PER;   // parts whose loads are in flight together
                    for (unsigned i0 = 0; i0 < others; i0 += AHEAD) {
                        float4 v[AHEAD][PER / 4];
                        float pm[AHEAD], pl[AHEAD];
#pragma unroll
                        for (int i = 0; i < AHEAD; ++i) {
                            const float *pp = part + (i0 + i) * P;
                            pm[i] = -INFINITY, pl[i] = 0.f;
                            if (i0 + i < others) {
                                pm[i] = __ldcg(pp + 8 * HD + mr);
                                pl[i] = __ldcg(pp + 8 * HD + 8 + mr);
#pragma unroll
                                for (int d = 0; d < PER / 4; ++d)
                                    v[i][d] = __ldcg(reinterpret_cast<const float4 *>(pp + mr * HD + md) + d);
                            }
                        }
                        float Mn = M;
#pragma unroll
                        for (int i = 0; i < AHEAD; ++i) Mn = fmaxf(Mn, pm[i]);
                        const float f0 = M == -INFINITY ? 0.f : ex2(M - Mn);
                        L = M == -INFINITY ? L : L * f0;
#pragma unroll
                        for (int d = 0; d < PER; ++d) acc[d] *= f0;
                        M = Mn;
#pragma unroll
                        for (int i = 0; i < AHEAD; ++i) {
                            if (i0 + i >= others) break;
                            const float f = pm[i] == -INFINITY ? 0.f : ex2(pm[i] - M);
                            L += pm[i] == -INFINITY ? pl[i] : f * pl[i];
#pragma unroll
                            for (int d = 0; d < PER / 4; ++d) {
                                acc[4 * d] = fmaf(f, v[i][d].x, acc[4 * d]);
                                acc[4 * d + 1] = fmaf(f, v[i][d].y, acc[4 * d + 1]);
                                acc[4 * d + 2] = fmaf(f, v[i][d].z, acc[4 * d + 2]);
                                acc[4 * d + 3] = fmaf(f, v[i][d].w, acc[4 * d + 3]);
                            }
                        }
                    }
                }
            }
            write_out();
        }
        u += end - cu.step;
        cu.step = end;
        if (u < u1) advance_item(cu);
        __syncthreads();   // merge and sh are free again
    }
    if (tell >= 0) told();
    // after a wait that ran out: the copies still in flight
    while (!ok && taken < issued) {
        mbar_wait_bounded(bars + (taken % NST) * 8, (taken / NST) & 1u, nullptr, kKvDrain);
        ++taken;
    }
}

// ---------------------------------------------------------------------------
// host side
// ---------------------------------------------------------------------------
// Workspace: the arrival counters (the part that stays zero between calls), then
// the partial results, one a CTA.
static constexpr int kMaxCtas = 512;
static constexpr size_t kCounterBytes = kMaxCtas * sizeof(int);
static_assert(kCounterBytes == TB_KV_WS_ZEROED, "the header's number");
size_t kv_attend_ws()
{
    size_t n = sizeof(float) * kMaxCtas * few_part(128);
    if (n < kManyCtas * kv_many_part_bytes()) n = kManyCtas * kv_many_part_bytes();
    if (n < kManyCtas * kv_tf32_part_bytes()) n = kManyCtas * kv_tf32_part_bytes();
    return kCounterBytes + n;
}

// Query rows per kv head up to which a sequence goes to k_kv_few, which passes over
// the cache once for 8 rows; the chunk kernels take as long for one row as for their
// tile.  Measured at 4096 positions, 8 kv heads of 128, 4 query heads each:
//                 1 sequence            16 sequences
//   rows        8    16   32   64       8    16    32    64
//   bf16 few   17    17   21   30      59    90   169   312   us
//        many  29    29   30   29      70    71    72    73
//   f32  few   20    27   41   64     125   232   441   848
//        tf32  65    65   64   63     195   196   197   199
//   f32 over bf16
//        few         19   25   36           108   203   390
//        tf32        64   62   62           147   148   150
// The crossing moves with the load (sequences x kv heads), from past 32 rows to past 8; a
// 16-bit cache under other activations, cheap in k_kv_few, leaves it at 16.
static int few_rows_of(bool narrow, long long load)
{
    return load < 24 ? 32 : load < 96 || narrow ? 16 : 8;
}

template <int HD, int TI, int TC>
static int few_launch(AttnArgs &a, int sms, cudaStream_t st)
{
    using Cfg = FewCfg<HD, TI, TC>;
    CUtensorMap km, vm;
    int ax[3];
    if (!kv_maps(a.c, HD, TC, kSlice, &km, &vm, ax)) return 0;
    a.ax_pos = ax[0], a.ax_head = ax[1], a.ax_page = ax[2];
    auto fn = k_kv_few<HD, TI, TC>;
    if (!smem_attr_once(reinterpret_cast<const void *>(fn), Cfg::SMEM)) {
        cudaGetLastError();
        return 0;
    }
    const int grid = sms * Cfg::CTAS < kMaxCtas ? sms * Cfg::CTAS : kMaxCtas;
    void *args[] = {&km, &vm, &a};
    return kv_launch(reinterpret_cast<const void *>(fn), dim3(grid), Cfg::W * 32, Cfg::SMEM, args, st);
}

template <int HD, int TI>
static int few_types(AttnArgs &a, int tc, int sms, cudaStream_t st)
{
    return tc == QT_F32   ? few_launch<HD, TI, QT_F32>(a, sms, st)
           : tc == QT_F16 ? few_launch<HD, TI, QT_F16>(a, sms, st)
                          : few_launch<HD, TI, QT_BF16>(a, sms, st);
}

template <int HD>
static int few(AttnArgs &a, int ti, int tc, int sms, cudaStream_t st)
{
    return ti == QT_F32   ? few_types<HD, QT_F32>(a, tc, sms, st)
           : ti == QT_F16 ? few_types<HD, QT_F16>(a, tc, sms, st)
                          : few_types<HD, QT_BF16>(a, tc, sms, st);
}

int kv_attend_launch(const KvView &c, const KvBatch &b, int hd, int ti, int tc, int nh, const KvRows &q,
                     const KvRows &o, float scale, int window, int sinks, int max_new, int max_len, void *ws, int *err,
                     int sms, uint32_t wait_limit, cudaStream_t st)
{
    const NvtxRange nvtx("tb.kv_attend");
    (void)max_len;
    AttnArgs a{c, b, q, o, nh, nh / c.n_kv_heads, window, sinks, scale * 1.4426950408889634f, err, wait_limit};
    a.arrived = static_cast<int *>(ws);
    a.part = reinterpret_cast<float *>(static_cast<char *>(ws) + kCounterBytes);
    a.many_rows = 0x7FFFFFFF;
    int before = 0;   // launches
    // Chunks go to the kernels with 128-row tiles: k_kv_many for 16-bit
    // activations over a cache of their type (whole tokens in 128 rows, a scale that
    // keeps the order of scores), k_kv_tf32 else.  Where the batch holds short
    // sequences besides, k_kv_few runs too and each takes its own; which sequences those
    // are is decided on the device.
    const bool many = ti == tc && tc != QT_F32 && scale > 0.f;
    const int rows = few_rows_of(!many && tc != QT_F32, static_cast<long long>(b.n_seqs) * c.n_kv_heads);
    if (a.group <= 128 && static_cast<long long>(max_new) * a.group > rows) {
        const bool mixed = b.n_tokens < static_cast<long long>(b.n_seqs) * max_new;
        const int few_rows = mixed ? rows : 0;
        int r = many ? kv_many_launch(a, hd, tc, few_rows, sms, st) : -1;
        if (r < 0) r = kv_tf32_launch(a, hd, ti, tc, few_rows, sms, st);
        if (r == 0 || !mixed) return r;
        a.many_rows = rows;
        before = 1;
    }
    const int r = hd == 128 ? few<128>(a, ti, tc, sms, st) : few<64>(a, ti, tc, sms, st);
    return r ? r + before : 0;
}

}  // namespace tb
