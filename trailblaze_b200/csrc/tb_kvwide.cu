// tb_kvwide.cu — attention of chunks of new tokens over the paged cache where the
// 16-bit tensor-core kernel does not apply (include/tb_gguf_dequant.h part 4): fp32
// activations over any cache, 16-bit activations over a cache of another type, and
// scales that are not positive.
//
// Items, units and the joining of parts are those of k_kv_many (tb_kvattn.cuh) with
// 128 query rows and tiles of 32 positions.  A CTA's 8 warps own 16 rows each and
// read the same K and V tiles, a TMA ring of 4 or 6 stages that the warps refill in turn,
// so the cache is read once for 128 rows.  The products and their splitting into
// parts of fewer bits are k_kv_few's: S^T = K Q^T, O^T += V^T P^T on mma.sync with
// the rows as two N = 8 tiles, so that K and V are fetched and split once for 16
// rows; tcgen05 has no operand wider than tf32 in fewer products, and its operands
// would first have to be written back to shared memory as parts.
//
// Measured (32 query and 8 kv heads of 128): 512 fp32 tokens at 1024 over an fp32
// cache in 144 us, over a bf16 cache in 84; the tensor pipe is busy for half of the
// fp32 time (three tf32 products for each), the rest is the splitting of K and V and
// what two warps a sub-core leave uncovered.
#include "tb_kvattn.cuh"

namespace tb {

static constexpr int kWTile = 32;      // positions of a tile
static constexpr int kWMin = 4;        // units of a CTA, at least
static constexpr int kWWarps = 8, kWThreads = kWWarps * 32;

struct WideArgs {
    AttnArgs a;
    int tpi;         // tokens of an item: 128 / G
    int few_rows;    // sequences of at most this many rows are another launch's
    int box;         // positions of one K or V box: 32 or 16
};

struct WideShared {
    KvScan scan;
    int fail, bad;
};

template <int HD, int TI, int TC>
struct WideCfg {
    static constexpr int ES = TC == QT_F32 ? 4 : 2;
    static constexpr int HALF = kWTile * HD * ES;      // K or V of a tile
    // fp32 caches: the low parts of Q live in shared memory, in the order of the
    // products (with both parts in registers 350 bytes a thread were spilled)
    static constexpr int QLO = TC == QT_F32 ? kWWarps * 2 * (HD / 8) * 32 * 8 : 0;
    static constexpr int NST = TC == QT_F32 ? 4 : 6;
    static constexpr int NQ = TC == QT_F32 ? 2 : TI == TC ? 1 : TC == QT_BF16 ? 3 : 2;
    static constexpr int NP = TC == QT_BF16 && TI == QT_F32 ? 3 : 2;
    static constexpr int SMEM = 1024 + NST * 2 * HALF + QLO + 2 * NST * 8 + static_cast<int>(sizeof(WideShared));
    static constexpr int PART = kWThreads * (HD / 2 + 8);   // floats of a partial result: O, m, l as the threads hold them
};

template <int HD, int TI, int TC>
__global__ void __launch_bounds__(kWThreads, 1)
    k_kv_wide(const __grid_constant__ CUtensorMap kmap, const __grid_constant__ CUtensorMap vmap,
              const __grid_constant__ WideArgs a)
{
    using Cfg = WideCfg<HD, TI, TC>;
    using I = typename KvType<TI>::E;
    using E = typename KvType<TC>::E;
    constexpr int NST = Cfg::NST, NQ = Cfg::NQ, NP = Cfg::NP, ES = Cfg::ES, NT = 2;
    constexpr bool X32 = TC == QT_F32;
    constexpr int KS = X32 ? HD / 8 : HD / 16;   // steps of the product over the head's dimensions
    constexpr int CB = HD * ES / 128;            // 128-byte columns of a row
    constexpr uint32_t kCol = kWTile * 128;
    extern __shared__ __align__(1024) uint8_t smraw[];
    uint8_t *sm = reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(smraw) + 1023) & ~uintptr_t(1023));
    uint2 *qlo = reinterpret_cast<uint2 *>(sm + NST * 2 * Cfg::HALF);   // [warp][nt][ks][lane]
    uint64_t *full = reinterpret_cast<uint64_t *>(sm + NST * 2 * Cfg::HALF + Cfg::QLO), *empty = full + NST;
    WideShared &sh = *reinterpret_cast<WideShared *>(empty + NST);
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, t = lane & 3;
    const AttnArgs &aa = a.a;
    const uint32_t lim = aa.wait_limit;
    int *err = aa.err;

    if (tid == 0) {
        for (int i = 0; i < NST; ++i) {
            mbar_init(smem_u32(full + i), 1);
            mbar_init(smem_u32(empty + i), kWWarps);
        }
        fence_mbar_init();
        sh.fail = 0;
        sh.bad = 0;
    }
    if (tid < 2) prefetch_map(tid ? &vmap : &kmap);
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    asm volatile("griddepcontrol.wait;" ::: "memory");
    KvCtaShare my;
    if (!kv_items_share<kWTile, kWMin, kWWarps, HD, I>(aa, a.tpi, a.few_rows, sh.scan, my)) return;
    __syncthreads();

    KvItem it = kv_item_first<kWTile>(aa, a.tpi, a.few_rows, sh.scan);
    int j0 = sh.scan.off;
    const uint32_t ring = smem_u32(sm), fb = smem_u32(full), eb = smem_u32(empty);
    const uint32_t n_tiles = static_cast<uint32_t>(my.u1 - my.u0);
    KvItem ic = it;            // the tile to be requested next
    int ij = j0;
    uint32_t issued = 0, taken = 0;
    bool ok = true;
    // Requests the next tile; the warp `turn` does it, the others keep count.  The
    // stage's last tile was taken two tiles ago, so the wait is short.
    auto issue = [&](int turn) {
        if (warp == turn && ok) {
            const uint32_t st = issued % NST, bar = fb + st * 8;
            if (issued >= NST) {
                ok = mbar_wait_bounded(eb + st * 8, (issued / NST - 1u) & 1u, err, lim);
                ok = __all_sync(0xFFFFFFFFu, ok);
                if (!ok) *reinterpret_cast<volatile int *>(&sh.fail) = 1;
            }
            if (ok) {
                const int p0 = kv_item_pos<kWTile>(ic, ij), boxes = kWTile / a.box, box = lane >> 1;
                int page = aa.c.n_pages, pos = 0;   // past the end: a page that reads as zeros
                const int p = p0 + box * a.box;
                if (box < boxes && p < ic.q.len) {
                    const uint32_t pi = fdiv(static_cast<uint32_t>(p), aa.c.page_div);
                    page = __ldg(aa.b.pages + static_cast<long long>(ic.s) * aa.b.pages_stride + pi);
                    pos = p - static_cast<int>(pi) * aa.c.page_size;
                    if (page < 0 || page >= aa.c.n_pages) {
                        atomicExch(err, ERR_RUNTIME);
                        *reinterpret_cast<volatile int *>(&sh.bad) = 1;
                        page = aa.c.n_pages;
                    }
                }
                const int y = aa.ax_pos == 0 ? pos : aa.ax_head == 0 ? ic.h : page;
                const int z = aa.ax_pos == 1 ? pos : aa.ax_head == 1 ? ic.h : page;
                const int w = aa.ax_pos == 2 ? pos : aa.ax_head == 2 ? ic.h : page;
                if (lane == 0) mbar_expect_tx(bar, 2 * Cfg::HALF);
                __syncwarp();
                if (box < boxes) {   // even lanes K, odd lanes V
                    const uint32_t dst = ring + st * 2 * Cfg::HALF + (lane & 1) * Cfg::HALF + box * a.box * 128;
#pragma unroll
                    for (int cb = 0; cb < CB; ++cb)
                        tma_load_4d(dst + cb * kCol, (lane & 1) ? &vmap : &kmap, cb * (128 / ES), y, z, w, bar);
                }
                __syncwarp();
            }
        }
        if (++issued < n_tiles && ++ij == ic.n) {
            ij = 0;
            kv_item_next<kWTile>(aa, a.tpi, a.few_rows, ic);
        }
    };

    unsigned long long u = my.u0;
    int tell = -1;   // the CTA that waits for this one's part
    auto told = [&]() {   // each warp for its stores
        __syncwarp();
        if (lane == 0) {
            __threadfence();
            atomicAdd(aa.arrived + tell, 1u);
        }
        __syncwarp();
        tell = -1;
    };
    const uint32_t krow = (lane & 7) + ((lane >> 3) & 1) * 8, kchunk = lane >> 4;   // ldmatrix rows of K
    const uint32_t vrow = (lane & 7) + (lane >> 4) * 8, vchunk = (lane >> 3) & 1;   // and of V, transposed
    while (u < my.u1) {
        const unsigned long long left = my.u1 - u;
        const int j1 = left < static_cast<unsigned>(it.n - j0) ? j0 + static_cast<int>(left) : it.n;
        const int p0 = it.q.len - it.q.n, rows = (it.t1 - it.t0) * aa.group, r0 = warp * 16;
        // rows g and g + 8 of the warp's 16 as the B operands; rows past the last are zero
        constexpr int NR = X32 ? 1 : NQ;   // parts in registers
        uint32_t qf[NT][NR][KS][2];
        float rs[NT][2];
        int pos[NT][2];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
            constexpr int QE = X32 ? 2 : 4;
            const int r = r0 + nt * 8 + g, tok = r / aa.group;
            const bool on = r < rows;
            const I *qp = static_cast<const I *>(aa.q.p) + (it.q.row0 + it.t0 + (on ? tok : 0)) * aa.q.row +
                          (it.h * aa.group + (on ? r - tok * aa.group : 0)) * aa.q.head;
            float rscale = aa.scale2;
            if constexpr (NQ == 1) {
#pragma unroll
                for (int ks = 0; ks < KS; ++ks)
#pragma unroll
                    for (int e = 0; e < 2; ++e)
                        qf[nt][0][ks][e] = on ? *reinterpret_cast<const uint32_t *>(qp + ks * 16 + 2 * t + 8 * e) : 0u;
            } else {
                float y[KS][QE], big = 0.f;
#pragma unroll
                for (int ks = 0; ks < KS; ++ks)
#pragma unroll
                    for (int e = 0; e < QE; ++e) {
                        y[ks][e] = on ? kv_f(qp[X32 ? ks * 8 + t + 4 * e : ks * 16 + 2 * t + 8 * (e >> 1) + (e & 1)]) : 0.f;
                        big = fmaxf(big, fabsf(y[ks][e]));
                    }
                if constexpr (X32) {
#pragma unroll
                    for (int ks = 0; ks < KS; ++ks) {
                        uint2 lo;
                        split_tf32(__float_as_uint(y[ks][0]), qf[nt][0][ks][0], lo.x);
                        split_tf32(__float_as_uint(y[ks][1]), qf[nt][0][ks][1], lo.y);
                        qlo[((warp * NT + nt) * KS + ks) * 32 + lane] = lo;   // read by this lane alone
                    }
                } else {
                    if constexpr (TC == QT_F16) {   // the row times 2^k, its largest element near 2^13
                        big = fmaxf(big, __shfl_xor_sync(0xFFFFFFFFu, big, 1));
                        big = fmaxf(big, __shfl_xor_sync(0xFFFFFFFFu, big, 2));
                        int k = 0;
                        if (big > 0.f && big < INFINITY) k = 13 - ilogbf(big);
                        k = max(-100, min(100, k));
                        const float up = ldexpf(1.f, k);
                        rscale = ldexpf(aa.scale2, -k);
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
                            for (int n = 0; n < NQ; ++n) qf[nt][n][ks][e] = pack16<TC>(y[ks][2 * e], y[ks][2 * e + 1]);
                }
            }
            // columns 2 t and 2 t + 1 of S^T and O^T
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                const int c = r0 + nt * 8 + 2 * t + e;
                pos[nt][e] = c < rows ? p0 + it.t0 + c / aa.group : -1;
                rs[nt][e] = __shfl_sync(0xFFFFFFFFu, rscale, (2 * t + e) * 4);
            }
        }
        if (issued == 0)
            for (uint32_t n = 0; n < NST && n < n_tiles; ++n) issue(n % kWWarps);
        const bool any = r0 < rows;   // this warp has rows
        const int pmin = p0 + it.t0 + r0 / aa.group, pmax = p0 + it.t0 + (min(r0 + 16, rows) - 1) / aa.group;
        float O[NT][HD / 16][4], m[NT][2], l[NT][2];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
            m[nt][0] = m[nt][1] = -INFINITY;
            l[nt][0] = l[nt][1] = 0.f;
#pragma unroll
            for (int i = 0; i < HD / 16; ++i)
#pragma unroll
                for (int e = 0; e < 4; ++e) O[nt][i][e] = 0.f;
        }

        for (int j = j0; j < j1; ++j) {
            const uint32_t st = taken % NST;
            ok = ok && mbar_wait_bounded(fb + st * 8, (taken / NST) & 1u, err, lim);
            ok = __all_sync(0xFFFFFFFFu, ok) && !*reinterpret_cast<volatile int *>(&sh.fail);
            if (!ok) *reinterpret_cast<volatile int *>(&sh.fail) = 1;
            uint32_t kb = ring + st * 2 * Cfg::HALF, vb = kb + Cfg::HALF;
            const int k0 = kv_item_pos<kWTile>(it, j);
            if (k0 + kWTile > it.q.len) {
                // the sequence's end: V past it, in the box that holds it, is zeroed: whatever
                // lies there, 0 * it has to be 0 (all warps pass here, in step)
                const int r1 = it.q.len - k0;
                for (int i = tid; i < (kWTile - r1) * (HD * ES / 16); i += kWThreads) {
                    const int r = r1 + i / (HD * ES / 16), c = i % (HD * ES / 16);
                    const uint32_t at = vb + (c >> 3) * kCol + r * 128 + ((c & 7) << 4);
                    if (ok) asm volatile("st.shared.v4.b32 [%0], {%1, %1, %1, %1};" ::"r"(at), "r"(0) : "memory");
                }
                fence_proxy_async_smem();   // before the stage's next copy
                __syncthreads();
            }
            kb = shared_after(kb);
            vb = shared_after(vb);
            const bool skip = !any || !ok || k0 > pmax ||
                              (aa.window > 0 && k0 + kWTile - 1 <= pmin - aa.window && k0 >= aa.sinks);
            if (!skip) {
#pragma unroll 1
                for (int s2 = 0; s2 < kWTile / 16; ++s2) {
                    const int js = k0 + s2 * 16;
                    if (js > pmax) break;
                    const uint32_t kr = s2 * 16 + krow, vr = s2 * 16 + vrow;
                    // ---- S^T = K Q^T, in short chains (see k_kv_few) ----
                    float c[NT][3][4];
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                        for (int i = 0; i < 3; ++i)
#pragma unroll
                            for (int e = 0; e < 4; ++e) c[nt][i][e] = 0.f;
#pragma unroll
                    for (int ks = 0; ks < KS; ++ks) {
                        const uint32_t ch = 2 * ks + kchunk;
                        uint32_t x[4];
                        ldsm4(kb + (ch >> 3) * kCol + kr * 128 + (((ch & 7) ^ (kr & 7)) << 4), x);
                        if constexpr (X32) {
                            uint32_t hi[4], lo[4];
#pragma unroll
                            for (int e = 0; e < 4; ++e) split_tf32(x[e], hi[e], lo[e]);
#pragma unroll
                            for (int nt = 0; nt < NT; ++nt) {
                                mma_tf32(c[nt][2], lo, qf[nt][0][ks][0], qf[nt][0][ks][1]);
                                mma_tf32(c[nt][ks & 1], hi, qf[nt][0][ks][0], qf[nt][0][ks][1]);
                            }
#pragma unroll
                            for (int nt = 0; nt < NT; ++nt) {
                                const uint2 lq = qlo[((warp * NT + nt) * KS + ks) * 32 + lane];
                                mma_tf32(c[nt][2], hi, lq.x, lq.y);
                            }
                        } else {
#pragma unroll
                            for (int n = NR - 1; n >= 0; --n)
#pragma unroll
                                for (int nt = 0; nt < NT; ++nt)
                                    mma16<TC>(c[nt][n > 0 ? 2 : ks & 1], x, qf[nt][n][ks][0], qf[nt][n][ks][1]);
                        }
                    }
                    const bool mask = js + 15 > pmin || (aa.window > 0 && js <= pmax - aa.window && js + 16 > aa.sinks);
                    float x[NT][4];
                    bool grow = false;
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
                        for (int e = 0; e < 4; ++e) x[nt][e] = ((c[nt][0][e] + c[nt][1][e]) + c[nt][2][e]) * rs[nt][e & 1];
                        if (mask) {
#pragma unroll
                            for (int e = 0; e < 4; ++e) {
                                const int jj = js + g + 8 * (e >> 1), p = pos[nt][e & 1];
                                const bool see = jj <= p && (aa.window == 0 || p - jj < aa.window || jj < aa.sinks);
                                x[nt][e] = see ? x[nt][e] : -INFINITY;
                            }
                        }
                        grow = grow || fmaxf(x[nt][0], x[nt][2]) > m[nt][0] + 8.f || fmaxf(x[nt][1], x[nt][3]) > m[nt][1] + 8.f;
                    }
                    if (__any_sync(0xFFFFFFFFu, grow)) {
#pragma unroll
                        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                            for (int e = 0; e < 2; ++e) {
                                float mx = fmaxf(x[nt][e], x[nt][e + 2]);
#pragma unroll
                                for (int o = 4; o < 32; o <<= 1) mx = fmaxf(mx, __shfl_xor_sync(0xFFFFFFFFu, mx, o));
                                mx = fmaxf(mx, m[nt][e]);
                                const float corr = m[nt][e] == -INFINITY ? 0.f : ex2(m[nt][e] - mx);
                                m[nt][e] = mx;
                                l[nt][e] *= corr;
#pragma unroll
                                for (int i = 0; i < HD / 16; ++i) O[nt][i][e] *= corr, O[nt][i][e + 2] *= corr;
                            }
                    }
                    // P^T: for X32 [8 positions][2 t and 2 t + 1 of them, row g], else 16-bit parts
                    uint32_t ph[NT][2][2], pl[NT][2][2], pb[NT][NP][2];
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
                        for (int e = 0; e < 4; ++e) x[nt][e] = ex2(x[nt][e] - (m[nt][e & 1] == -INFINITY ? 0.f : m[nt][e & 1]));
                        l[nt][0] += x[nt][0] + x[nt][2];
                        l[nt][1] += x[nt][1] + x[nt][3];
                        if constexpr (X32) {
#pragma unroll
                            for (int kb8 = 0; kb8 < 2; ++kb8)
#pragma unroll
                                for (int e = 0; e < 2; ++e) {
                                    const int from = (2 * t + e) * 4 + (g >> 1);
                                    const float y0 = __shfl_sync(0xFFFFFFFFu, x[nt][2 * kb8], from);
                                    const float y1 = __shfl_sync(0xFFFFFFFFu, x[nt][2 * kb8 + 1], from);
                                    split_tf32(__float_as_uint((g & 1) ? y1 : y0), ph[nt][kb8][e], pl[nt][kb8][e]);
                                }
                        } else {
#pragma unroll
                            for (int n = 0; n < NP; ++n)
#pragma unroll
                                for (int e = 0; e < 2; ++e) pb[nt][n][e] = mat_t(pack16<TC>(x[nt][2 * e], x[nt][2 * e + 1]));
                        }
                    }
                    // ---- O^T += V^T P^T, each slice's sum added in fp32 ----
                    if constexpr (X32) {
#pragma unroll
                        for (int jb = 0; jb < HD / 64; ++jb) {
                            uint4 v[2][2][2];   // [8 positions][column 2 jb, 2 jb + 1][position 2 t, 2 t + 1]: 4 dimensions each
#pragma unroll
                            for (int kb8 = 0; kb8 < 2; ++kb8)
#pragma unroll
                                for (int cc = 0; cc < 2; ++cc)
#pragma unroll
                                    for (int e = 0; e < 2; ++e) {
                                        const uint32_t r = s2 * 16 + kb8 * 8 + 2 * t + e;
                                        v[kb8][cc][e] = lds_u128(vb + (2 * jb + cc) * kCol + r * 128 + ((g ^ (r & 7)) << 4));
                                    }
#pragma unroll
                            for (int d = 0; d < 4; ++d) {
                                float o[NT][4];
#pragma unroll
                                for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                                    for (int e = 0; e < 4; ++e) o[nt][e] = 0.f;
#pragma unroll
                                for (int kb8 = 0; kb8 < 2; ++kb8) {
                                    uint32_t hi[4], lo[4];
#pragma unroll
                                    for (int e = 0; e < 4; ++e) {
                                        const uint4 &w = v[kb8][e & 1][e >> 1];
                                        split_tf32(d == 0 ? w.x : d == 1 ? w.y : d == 2 ? w.z : w.w, hi[e], lo[e]);
                                    }
#pragma unroll
                                    for (int nt = 0; nt < NT; ++nt) mma_tf32(o[nt], lo, ph[nt][kb8][0], ph[nt][kb8][1]);
#pragma unroll
                                    for (int nt = 0; nt < NT; ++nt) mma_tf32(o[nt], hi, pl[nt][kb8][0], pl[nt][kb8][1]);
#pragma unroll
                                    for (int nt = 0; nt < NT; ++nt) mma_tf32(o[nt], hi, ph[nt][kb8][0], ph[nt][kb8][1]);
                                }
#pragma unroll
                                for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                                    for (int e = 0; e < 4; ++e) O[nt][jb * 4 + d][e] += o[nt][e];
                            }
                        }
                    } else {
#pragma unroll
                        for (int i = 0; i < HD / 16; ++i) {
                            const uint32_t ch = 2 * i + vchunk;
                            uint32_t v[4];
                            ldsm4t(vb + (ch >> 3) * kCol + vr * 128 + (((ch & 7) ^ (vr & 7)) << 4), v);
                            float o[NT][4];
#pragma unroll
                            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                                for (int e = 0; e < 4; ++e) o[nt][e] = 0.f;
#pragma unroll
                            for (int n = NP - 1; n >= 0; --n)
#pragma unroll
                                for (int nt = 0; nt < NT; ++nt) mma16<TC>(o[nt], v, pb[nt][n][0], pb[nt][n][1]);
#pragma unroll
                            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                                for (int e = 0; e < 4; ++e) O[nt][i][e] += o[nt][e];
                        }
                    }
                }
            }
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                for (int i = 0; i < HD / 16; ++i) pin(O[nt][i]);
            __syncwarp();   // every lane has read the stage
            if (lane == 0) mbar_arrive(eb + st * 8);
            ++taken;
            if (taken >= 2 && issued < n_tiles) issue(taken % kWWarps);   // into the stage of the tile before
            if (tell >= 0) told();
        }
        // ---- the item, or this CTA's part of it ----
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int e = 0; e < 2; ++e)
#pragma unroll
                for (int o = 4; o < 32; o <<= 1) l[nt][e] += __shfl_xor_sync(0xFFFFFFFFu, l[nt][e], o);
        if (j0 > 0) {
            // not the item's beginning: the part goes to the CTA that has it, as the threads hold it
            // (a page outside the pool: as NaN, so that the rows are done again there)
            const bool bad = *reinterpret_cast<volatile int *>(&sh.bad) != 0;
            float4 *mp = reinterpret_cast<float4 *>(aa.part + static_cast<size_t>(my.cta) * Cfg::PART) + tid;
#pragma unroll
            for (int nt = 0; nt < NT && any; ++nt) {   // warps without rows stay out of the traffic
#pragma unroll
                for (int i = 0; i < HD / 16; ++i)
                    __stcg(mp + (nt * (HD / 16) + i) * kWThreads, make_float4(O[nt][i][0], O[nt][i][1], O[nt][i][2], O[nt][i][3]));
                __stcg(mp + (NT * (HD / 16) + nt) * kWThreads, 
                       bad ? make_float4(m[nt][0], m[nt][1], NAN, NAN) : make_float4(m[nt][0], m[nt][1], l[nt][0], l[nt][1]));
            }
            tell = static_cast<int>(my.share.of(u - j0));
        } else {
            bool odd[NT][2];
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) odd[nt][0] = odd[nt][1] = *reinterpret_cast<volatile int *>(&sh.bad) != 0;
            if (j1 < it.n) {
                // the beginning: the other parts, of the CTAs after this one, in order (waited for, as
                // every wait, within a limit: those CTAs were started before this one)
                const unsigned others = my.share.of(u + it.n - 1) - my.cta;
                uint32_t i = 0;
                unsigned n = 0;
                do {
                    asm volatile("ld.acquire.gpu.global.u32 %0, [%1];" : "=r"(n) : "l"(aa.arrived + my.cta) : "memory");
                } while (n < kWWarps * others && ++i < lim && !*reinterpret_cast<volatile int *>(&sh.fail));
                if (n < kWWarps * others) {
                    if (!*reinterpret_cast<volatile int *>(&sh.fail)) atomicExch(err, ERR_WAIT_TIMEOUT);
                    *reinterpret_cast<volatile int *>(&sh.fail) = 1;
                }
                __syncthreads();                        // every warp has seen the count
                if (tid == 0) aa.arrived[my.cta] = 0;   // zero between calls
                for (unsigned c = 0; c < others && any; ++c) {
                    const float4 *pp = reinterpret_cast<const float4 *>(aa.part + static_cast<size_t>(my.cta + 1 + c) * Cfg::PART) + tid;
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt) {
                        const float4 ml = __ldcg(pp + (NT * (HD / 16) + nt) * kWThreads);
                        const float pm[2] = {ml.x, ml.y}, pl[2] = {ml.z, ml.w};
                        float f0[2], f1[2];
#pragma unroll
                        for (int e = 0; e < 2; ++e) {
                            const float mx = fmaxf(m[nt][e], pm[e]);
                            f0[e] = m[nt][e] == -INFINITY ? 0.f : ex2(m[nt][e] - mx);
                            f1[e] = pm[e] == -INFINITY ? 0.f : ex2(pm[e] - mx);
                            // nothing seen: l is 0, unless what was seen was NaN
                            l[nt][e] = (m[nt][e] == -INFINITY ? l[nt][e] : l[nt][e] * f0[e]) + (pm[e] == -INFINITY ? pl[e] : pl[e] * f1[e]);
                            m[nt][e] = mx;
                        }
#pragma unroll
                        for (int i2 = 0; i2 < HD / 16; ++i2) {
                            const float4 v = __ldcg(pp + (nt * (HD / 16) + i2) * kWThreads);
                            O[nt][i2][0] = O[nt][i2][0] * f0[0] + v.x * f1[0];
                            O[nt][i2][1] = O[nt][i2][1] * f0[1] + v.y * f1[1];
                            O[nt][i2][2] = O[nt][i2][2] * f0[0] + v.z * f1[0];
                            O[nt][i2][3] = O[nt][i2][3] * f0[1] + v.w * f1[1];
                        }
                    }
                }
            }
            I *out = static_cast<I *>(const_cast<void *>(aa.o.p));
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    const int r = r0 + nt * 8 + 2 * t + e, tok = r / aa.group;
                    const float inv = l[nt][e] == 0.f ? 0.f : 1.0f / l[nt][e];
                    bool bad = odd[nt][e] || !isfinite(l[nt][e]) || m[nt][e] == INFINITY;
                    float nil = 0.f;
#pragma unroll
                    for (int i = 0; i < HD / 16; ++i) nil = fmaf(O[nt][i][e], 0.f, fmaf(O[nt][i][e + 2], 0.f, nil));
                    bad = bad || nil != 0.f || isnan(nil);
#pragma unroll
                    for (int o = 4; o < 32; o <<= 1) bad = __shfl_xor_sync(0xFFFFFFFFu, static_cast<int>(bad), o) || bad;
                    odd[nt][e] = bad;
                    if (r >= rows) continue;
                    I *op = out + (it.q.row0 + it.t0 + tok) * aa.o.row + (it.h * aa.group + (r - tok * aa.group)) * aa.o.head;
#pragma unroll
                    for (int k = 0; k < 2; ++k)
                        if constexpr (X32) {
#pragma unroll
                            for (int jb = 0; jb < HD / 64; ++jb) {
                                alignas(16) I v[4];
#pragma unroll
                                for (int d = 0; d < 4; ++d) kv_store1(v + d, O[nt][jb * 4 + d][e + 2 * k] * inv);
                                I *q = op + jb * 64 + k * 32 + 4 * g;
                                if constexpr (sizeof(I) == 4) *reinterpret_cast<float4 *>(q) = *reinterpret_cast<const float4 *>(v);
                                else *reinterpret_cast<uint2 *>(q) = *reinterpret_cast<const uint2 *>(v);
                            }
                        } else {
#pragma unroll
                            for (int i = 0; i < HD / 16; ++i) kv_store1(op + i * 16 + k * 8 + g, O[nt][i][e + 2 * k] * inv);
                        }
                }
            // rows that are not finite: V of a position that a row does not see may have been
            // (0 * NaN), or a page lies outside the pool.  Once more, over their own positions only.
            __syncwarp();
#pragma unroll 1
            for (int r = 0; r < 16; ++r) {
                const bool b0 = r & 1 ? (r & 8 ? odd[1][1] : odd[0][1]) : (r & 8 ? odd[1][0] : odd[0][0]);
                if (!__shfl_sync(0xFFFFFFFFu, static_cast<int>(b0), (r & 7) >> 1) || r0 + r >= rows || !ok) continue;
                constexpr int D = HD / 32;
                const int tok = (r0 + r) / aa.group, hh = (r0 + r) - tok * aa.group;
                const I *qp = static_cast<const I *>(aa.q.p) + (it.q.row0 + it.t0 + tok) * aa.q.row +
                              (it.h * aa.group + hh) * aa.q.head + lane * D;
                float q[D], rm, rl, acc[D];
#pragma unroll
                for (int d = 0; d < D; ++d) q[d] = kv_f(qp[d]) * aa.scale2;
                kv_row_attend<HD, E>(aa.b, aa.c, it.s, it.h, p0 + it.t0 + tok, 0, it.q.len, aa.window, aa.sinks, q, rm, rl,
                                     acc, err);
                I *op = out + (it.q.row0 + it.t0 + tok) * aa.o.row + (it.h * aa.group + hh) * aa.o.head + lane * D;
#pragma unroll
                for (int d = 0; d < D; ++d) kv_store1(op + d, rl == 0.f ? 0.f : acc[d] / rl);
                __syncwarp();
            }
        }
        u += j1 - j0;
        j0 = 0;
        if (u < my.u1) kv_item_next<kWTile>(aa, a.tpi, a.few_rows, it);
    }
    if (tell >= 0) told();
    // after a wait that ran out: the copies still in flight, as far as they come
    __syncthreads();
    if (sh.fail && warp == 0)
        for (uint32_t n = issued > NST ? issued - NST : 0; n < issued; ++n)
            mbar_wait_bounded(fb + (n % NST) * 8, (n / NST) & 1u, err, lim);
}

// ---------------------------------------------------------------------------
// host side
// ---------------------------------------------------------------------------
size_t kv_wide_part_bytes() { return sizeof(float) * WideCfg<128, QT_F32, QT_F32>::PART; }

template <int HD, int TI, int TC>
static int wide_launch(WideArgs &w, int sms, cudaStream_t st)
{
    AttnArgs &a = w.a;
    CUtensorMap km, vm;
    int ax[3];
    w.box = a.c.page_size % 32 ? 16 : 32;
    if (!kv_maps(a.c, HD, TC, w.box, &km, &vm, ax)) return 0;
    a.ax_pos = ax[0], a.ax_head = ax[1], a.ax_page = ax[2];
    auto fn = k_kv_wide<HD, TI, TC>;
    if (!smem_attr_once(reinterpret_cast<const void *>(fn), WideCfg<HD, TI, TC>::SMEM)) {
        cudaGetLastError();
        return 0;
    }
    void *args[] = {&km, &vm, &w};
    return kv_launch(reinterpret_cast<const void *>(fn), dim3(sms < kManyCtas ? sms : kManyCtas), kWThreads,
                     WideCfg<HD, TI, TC>::SMEM, args, st);
}

template <int HD, int TI>
static int wide_types(WideArgs &w, int tc, int sms, cudaStream_t st)
{
    return tc == QT_F32   ? wide_launch<HD, TI, QT_F32>(w, sms, st)
           : tc == QT_F16 ? wide_launch<HD, TI, QT_F16>(w, sms, st)
                          : wide_launch<HD, TI, QT_BF16>(w, sms, st);
}

template <int HD>
static int wide_hd(WideArgs &w, int ti, int tc, int sms, cudaStream_t st)
{
    return ti == QT_F32   ? wide_types<HD, QT_F32>(w, tc, sms, st)
           : ti == QT_F16 ? wide_types<HD, QT_F16>(w, tc, sms, st)
                          : wide_types<HD, QT_BF16>(w, tc, sms, st);
}

int kv_wide_launch(AttnArgs a, int hd, int ti, int tc, int few_rows, int sms, cudaStream_t st)
{
    WideArgs w{a, 128 / a.group, few_rows, 0};
    return hd == 128 ? wide_hd<128>(w, ti, tc, sms, st) : wide_hd<64>(w, ti, tc, sms, st);
}

}  // namespace tb
