// Forward kernel of the sliding-window attention, and of the shared prefix of a decoding
// batch, for sm_100a (included by window_sm100.cu inside namespace bfk).
//
// Window mode (kPartial = false). Query i of head h stands at position p = i + n_kv - n_q
// and sees the keys j <= p with j > p - window or j < sinks, of KV head h / group:
//   O_i = sum_j softmax_j(scale q_i.k_j) v_j,   lse_i = log sum_j exp(scale q_i.k_j).
// A query that sees no key gets O = 0 and lse = -inf.
// Partial mode (kPartial = true). All query rows of a KV head (batch x group x tokens)
// against one range of the prefix's KV tiles, nothing masked; fp32 O normalised over that
// range and its log2-sum-exp2, joined later.
//
// The roles, TMEM use and softmax are those of the dense kernels beside it (16 softmax
// warps with two threads per row, a TMA producer, issuers, persistent CTAs). What differs:
//   * an item is two 128-row query tiles of one KV head, each with a list of KV tiles of
//     its own. With an even group the two are two heads at the same rows, so both lists
//     are the same and K/V are read once for both; otherwise they are two consecutive row
//     blocks, and a tile sits out the steps that only the other one needs;
//   * up to 32 sinks (kNarrow) the step of the sink tile is 32 columns wide: it comes
//     first, so it has no maximum to compare with and nothing to rescale;
//   * the list is the sink tiles [0, ns) and then the window's tiles [lo, hi), so the work
//     of a row is proportional to the keys that it sees and not to the length;
//   * a tile may be wholly masked for some of its rows (the window's lower edge, rows
//     before the first key), so the running maximum may stay -inf for some steps;
//   * bf16 or fp16. In fp16, P is scaled by 2^7: its entries then lie in [0, 2^15] (2^8 of
//     the lazy rescale times 2^7), below fp16's 65504, and the smallest kept entry is
//     2^-31 of the largest instead of 2^-24.
// Tensor maps are 4-D with the caller's strides; rows past the end read as zero.
namespace win {

constexpr int kSoftWarps = 16;     // 8 per query tile
constexpr int kProducerWarp = 16;  // TMA producer
constexpr int kSWarp = 17;         // issues S = Q K^T of query tile 0, warp 19 of tile 1; owns the TMEM allocation
constexpr int kPVWarp = 18;        // issues O += P V
constexpr int kThreads = 20 * 32;
constexpr int kTmemCols = 512;
// Launch budget 96 x 640 = 61440 registers: 104 x 512 + 64 x 128.
constexpr int kSoftRegs = 104, kIssueRegs = 64;
static_assert(kSoftRegs * 512 + kIssueRegs * 128 <= 96 * kThreads, "register split exceeds the launch budget");

template <int D>
struct Cfg {
    static constexpr int kChunks = D / 64;
    static constexpr int kChunkBytes = 128 * 64 * 2;
    static constexpr int kTile = kChunks * kChunkBytes;
    // d = 64 leaves room for two query buffers and a four-deep K/V ring; at d = 128 one
    // query buffer and two stages fill shared memory.
    static constexpr int kStages = D == 64 ? 4 : 2;
    static constexpr int kQBufs = D == 64 ? 2 : 1;
    static constexpr int kOffQ = 0;  // [kQBufs][2 tiles]
    static constexpr int kOffK = kOffQ + kQBufs * 2 * kTile;
    static constexpr int kOffV = kOffK + kStages * kTile;
    static constexpr int kOffBar = kOffV + kStages * kTile;
    // TMEM: S0 S1 | P0 P1 | O0 O1 at d = 64; at d = 128 O fills the second half and P is
    // written over the lower half of S.
    static constexpr bool kSepP = D == 64;
    static constexpr int kColP = kSepP ? 256 : 0;
    static constexpr int kStepP = kSepP ? 64 : 128;
    static constexpr int kColO = kSepP ? 384 : 256;
};

template <int D>
struct Bars {
    uint64_t q_full[Cfg<D>::kQBufs][2];
    uint64_t q_empty[Cfg<D>::kQBufs];
    uint64_t k_full[Cfg<D>::kStages];
    uint64_t k_empty[Cfg<D>::kStages];
    uint64_t v_full[Cfg<D>::kStages];
    uint64_t v_empty[Cfg<D>::kStages];
    uint64_t s_full[2];  // the next three follow it: the softmax warps address them from here
    uint64_t s_empty[2];
    uint64_t p_full[2];
    uint64_t pv_done[2];
    uint64_t drain[3];
    uint32_t tmem_base;
    int abort_flag;
};

template <int D>
constexpr int smem_bytes() {
    return Cfg<D>::kOffBar + (int)sizeof(Bars<D>) + 1024;
}
static_assert(smem_bytes<64>() <= 227 * 1024 && smem_bytes<128>() <= 227 * 1024, "shared memory");

enum : unsigned {
    kSiteProdQ = 0x700,
    kSiteProdK = 0x701,
    kSiteProdV = 0x702,
    kSiteMmaQ = 0x710,  // + t
    kSiteMmaK = 0x720,  // +0 K full, +1 + t PV_t done, +3 + t S_t loaded
    kSiteMmaV = 0x730,  // +0 V full, +1 + t P_t full
    kSiteSoftS = 0x740,
    kSiteSoftPV = 0x741,
};

// n / d by a product, for 0 <= n < 2^31 and d >= 1: with l = ceil(log2 d) and
// m = floor(2^32 (2^l - d) / d) + 1, n / d = (floor(m n / 2^32) + n) >> l (Granlund and
// Montgomery 1994).
struct FastDiv {
    uint32_t m, l;
    void set(uint32_t d) {
        for (l = 0; (1ull << l) < d; ++l) {}
        m = (uint32_t)(((1ull << 32) * ((1ull << l) - d)) / d + 1);
    }
    __device__ __forceinline__ int operator()(int n) const { return (int)((__umulhi(m, (uint32_t)n) + (uint32_t)n) >> l); }
};

struct Params {
    int items;
    int batch, hq, hkv, group;
    int n_q, n_kv;
    int nk;          // KV tiles
    float scale_log2;
    void* out;       // [B, Hq, n_q, D] bf16 / fp16; partial mode: fp32 [splits][rows][D]
    float* lse;      // [B, Hq, n_q] natural log, optional; partial mode: [splits][rows] log2
    unsigned long long timeout_ns;
    // window mode
    int window, sinks, ns;  // window clamped to n_kv, sinks, sink tiles
    FastDiv by_units, by_heads, by_group;
    int q_blocks;           // item blocks along the queries
    int pair_heads;         // the two tiles are two heads of a group
    // partial mode
    int q_rows;             // group * tokens: rows of one (sequence, KV head)
    int seqs_per_tile;      // whole sequences in a 128-row tile, 0: a sequence spans several tiles
    int tiles_per_seq;      // 128-row tiles of a sequence where seqs_per_tile == 0
    int row_tiles;          // 128-row query tiles of a KV head
    int pairs;              // ceil(row_tiles / 2)
    int split_tiles;        // KV tiles of a split
    long long rows;         // batch * hq * tokens
};

// What an item's two tiles are and which KV tiles they see.
struct Item {
    int b[2], head[2], row0[2];  // window mode: batch, query head, first row; partial: first sequence, -, first row
    int kvh, kvb, split;
    int lo[2], hi[2];            // window tiles of query tile t; hi = 0: the tile is idle
    int j_lo, n_sink, steps;     // the steps of both: tiles [0, n_sink), then from j_lo on
};

template <bool kPartial>
__device__ __forceinline__ void decode(const Params& p, int item, Item& it) {
    if constexpr (kPartial) {
        const int pr = item % p.pairs;
        const int rest = item / p.pairs;
        it.kvh = rest % p.hkv;
        it.split = rest / p.hkv;
        it.kvb = 0;
        const int j0 = it.split * p.split_tiles, j1 = min(j0 + p.split_tiles, p.nk);
#pragma unroll
        for (int t = 0; t < 2; ++t) {
            const int u = 2 * pr + t;
            it.head[t] = 0;
            it.b[t] = p.seqs_per_tile ? u * p.seqs_per_tile : u / p.tiles_per_seq;
            it.row0[t] = p.seqs_per_tile ? 0 : (u % p.tiles_per_seq) * 128;
            it.lo[t] = j0;
            it.hi[t] = u < p.row_tiles ? j1 : 0;
        }
        it.j_lo = j0;
        it.n_sink = 0;
        it.steps = j1 - j0;
    } else {
        const int per_head = p.pair_heads ? p.hq / 2 : p.hq;
        const int units = p.batch * per_head;
        // Late rows see the most keys: they are handed out first.
        const int late = p.by_units(item), unit = item - late * units;
        const int qb = p.q_blocks - 1 - late;
        const int b = p.by_heads(unit), hu = unit - b * per_head;
        it.split = 0;
        it.kvb = b;
        it.kvh = p.by_group(p.pair_heads ? 2 * hu : hu);
        const int off = p.n_kv - p.n_q;
        int lo_u = p.nk, hi_u = 0;
#pragma unroll
        for (int t = 0; t < 2; ++t) {
            it.b[t] = b;
            it.head[t] = p.pair_heads ? 2 * hu + t : hu;
            it.row0[t] = p.pair_heads ? qb * 128 : qb * 256 + t * 128;
            const int p_first = it.row0[t] + off;
            const int p_last = min(it.row0[t] + 128, p.n_q) - 1 + off;
            it.lo[t] = max(0, p_first - p.window + 1) >> 7;
            it.hi[t] = it.row0[t] < p.n_q && p_last >= 0 ? (p_last >> 7) + 1 : 0;
            if (it.hi[t] > 0) {
                lo_u = min(lo_u, it.lo[t]);
                hi_u = max(hi_u, it.hi[t]);
            }
        }
        it.j_lo = lo_u;
        it.n_sink = hi_u > 0 ? min(p.ns, lo_u) : 0;
        it.steps = hi_u > 0 ? it.n_sink + hi_u - lo_u : 0;
    }
}

// Bits 0 .. n - 1 (none for n <= 0, all for n >= 32).
__device__ __forceinline__ uint32_t below(int n) {
    return n >= 32 ? ~0u : (1u << max(n, 0)) - 1u;
}

// a[t] for the two-entry arrays of an Item, which stay in registers.
template <typename T>
__device__ __forceinline__ T pick(const T (&a)[2], int t) {
    return t ? a[1] : a[0];
}
__device__ __forceinline__ int step_tile(const Item& it, int s) { return s < it.n_sink ? s : it.j_lo + s - it.n_sink; }
__device__ __forceinline__ bool sees(const Params& p, const Item& it, int t, int j) {
    return j < pick(it.hi, t) && (j >= pick(it.lo, t) || j < p.ns);
}

template <int D, bool kF16, bool kPartial, bool kNarrow>
__global__ void __launch_bounds__(kThreads, 1)
    window_fwd_kernel(const __grid_constant__ CUtensorMap tmQ, const __grid_constant__ CUtensorMap tmK,
                      const __grid_constant__ CUtensorMap tmV, const Params p) {
    using C = Cfg<D>;
    extern __shared__ uint8_t smem_raw[];
    uint8_t* smem = align1024(smem_raw);
    Bars<D>* bars = reinterpret_cast<Bars<D>*>(smem + C::kOffBar);
    const int warp = __shfl_sync(0xffffffffu, (int)(threadIdx.x >> 5), 0);  // known to be uniform
    const int lane = threadIdx.x & 31;

    if (threadIdx.x == 0) {
        for (int b = 0; b < C::kQBufs; ++b) {
            mbar_init(smem_addr(&bars->q_full[b][0]), 1);
            mbar_init(smem_addr(&bars->q_full[b][1]), 1);
            mbar_init(smem_addr(&bars->q_empty[b]), 2);  // one arrival per S issuer
        }
        for (int s = 0; s < C::kStages; ++s) {
            mbar_init(smem_addr(&bars->k_full[s]), 1);
            mbar_init(smem_addr(&bars->k_empty[s]), 2);
            mbar_init(smem_addr(&bars->v_full[s]), 1);
            mbar_init(smem_addr(&bars->v_empty[s]), 1);
        }
        for (int t = 0; t < 2; ++t) {
            mbar_init(smem_addr(&bars->s_full[t]), 1);
            mbar_init(smem_addr(&bars->s_empty[t]), 8);  // one arrival per softmax warp of the tile
            mbar_init(smem_addr(&bars->p_full[t]), 8);
            mbar_init(smem_addr(&bars->pv_done[t]), 1);
        }
        for (int r = 0; r < 3; ++r) mbar_init(smem_addr(&bars->drain[r]), 1);
        bars->abort_flag = 0;
        fence_barrier_init();
    }
    if (warp == kProducerWarp && lane == 0) {
        tma_prefetch_desc(&tmQ);
        tma_prefetch_desc(&tmK);
        tma_prefetch_desc(&tmV);
    }
    if (warp == kSWarp) {
        tmem_alloc(smem_addr(&bars->tmem_base), kTmemCols);
        tmem_relinquish();
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = bars->tmem_base;
    const WaitCtl ctl{&bars->abort_flag, &g_wait_status, p.timeout_ns};
    // Nothing above touches global data: it overlaps the previous grid's tail. In partial mode
    // the next grid is the cache's part of the step, which reads nothing of this one: it may
    // start, and use the multiprocessors that this grid leaves free, as soon as the grids
    // before this one are complete.
    if (!kPartial) griddep_launch_dependents();
    griddep_wait();
    if (kPartial) griddep_launch_dependents();

    if (warp < kSoftWarps)
        regs_inc<kSoftRegs>();
    else
        regs_dec<kIssueRegs>();

    if (warp < kSoftWarps) {
        // ------------------------------------------------------------ softmax
        // Warp w of tile t covers 16 TMEM lanes; lanes i and i + 16 share a row, one per
        // 64-column half of S.
        const int t = warp >> 3;
        const int quarter = warp & 3;
        const int sub = (warp >> 2) & 1;
        const int h = lane >> 4;
        const int row = quarter * 32 + sub * 16 + (lane & 15);
        const uint32_t lane_off = (uint32_t)(quarter * 32 + sub * 16) << 16;
        const uint32_t tS = tmem + lane_off + (uint32_t)(t * 128);
        const uint32_t tP = C::kSepP ? tmem + lane_off + (uint32_t)(C::kColP + t * C::kStepP) : tS;
        const uint32_t tO = C::kSepP ? tP + (uint32_t)(C::kColO - C::kColP) : tS + C::kColO;
        const uint64_t sl2_2 = f2_pack(p.scale_log2, p.scale_log2);
        // s_full, s_empty, p_full and pv_done of tile t, two barriers of 8 bytes each apart.
        const uint32_t bar_s = smem_addr(&bars->s_full[t]);
        const uint32_t bar_se = bar_s + 16, bar_p = bar_s + 32, bar_pv = bar_s + 48;
        constexpr float kShift = kF16 ? 7.f : 0.f;  // P is scaled by 2^kShift
        uint32_t g = 0;  // steps of this tile so far
        bool ok = true;

        for (int item = blockIdx.x; item < p.items && ok; item += gridDim.x) {
            // This tile's own steps, in the order of the item's: sink tiles, then the window's.
            int n_sink, skip, steps, pos;
            {
                Item it;
                decode<kPartial>(p, item, it);
                const int lo = pick(it.lo, t), hi = pick(it.hi, t);
                n_sink = min(p.ns, lo);
                skip = lo - n_sink;
                steps = hi > 0 ? hi - skip : 0;
                pos = pick(it.row0, t) + row + p.n_kv - p.n_q;
            }
            float m_use = -INFINITY;  // log2-domain maximum that P, O and l refer to
            float l_half = 0.f;       // row sum over this thread's column half

            if (kNarrow && n_sink > 0 && steps > 0) {
                // The sinks' step, 32 columns: this thread's are 16 h .. 16 h + 15. Every row of the
                // tile is past the sinks (lo > 0) and sees them all.
                if (!(ok = warp_wait(bar_s, g & 1u, ctl, kSiteSoftS))) break;
                tc_fence_after();
                uint32_t s[16], pk[8];
                tmem_ld16x32bx2_x16<16>(tS, s);
                tmem_wait_ld();
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(bar_se);
                float mx = -INFINITY;
#pragma unroll
                for (int c = 0; c < 16; ++c) {
                    if (c >= p.sinks - h * 16) s[c] = __float_as_uint(-INFINITY);
                    mx = fmaxf(mx, __uint_as_float(s[c]));
                }
                mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 16));
                m_use = mx * p.scale_log2;
                const float neg_m = m_use == -INFINITY ? 0.f : kShift - m_use;
#pragma unroll
                for (int c = 0; c < 16; c += 2) {
                    const float p0 = fast_exp2(fmaf(__uint_as_float(s[c]), p.scale_log2, neg_m));
                    const float p1 = fast_exp2(fmaf(__uint_as_float(s[c + 1]), p.scale_log2, neg_m));
                    l_half += p0 + p1;
                    pk[c / 2] = kF16 ? pack_f16x2(p0, p1) : pack_bf16x2(p0, p1);
                }
                if (C::kSepP && g > 0) {
                    if (!(ok = warp_wait(bar_pv, (g - 1) & 1u, ctl, kSiteSoftPV))) break;
                    tc_fence_after();
                }
                tmem_st16x32bx2_x8<8>(tP, pk);
                tmem_wait_st();
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(bar_p);
                ++g;
            }
            for (int s_i = kNarrow ? n_sink : 0; s_i < steps; ++s_i, ++g) {
                const int j = s_i < n_sink ? s_i : s_i + skip;
                if (!(ok = warp_wait(bar_s, g & 1u, ctl, kSiteSoftS))) break;
                tc_fence_after();
                uint32_t s[2][32];
                tmem_ld16x32bx2_x32<64>(tS + 0, s[0]);
                tmem_ld16x32bx2_x32<64>(tS + 32, s[1]);
                tmem_wait_ld();
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(bar_se);  // S_t is in registers

                const int c0 = j * 128 + h * 64;
                // Seen: column c with c < last, and c >= first or c < snk. As a word of bits per 32
                // columns a column costs two instructions, not the four of the comparisons (which
                // took as long as the exponentials: two or three steps of an item are masked).
                const int last = kPartial ? p.n_kv - c0 : pos + 1 - c0;
                const int first = kPartial ? 0 : pos + 1 - p.window - c0;
                const int snk = kPartial ? 0 : p.sinks - c0;
                if (last < 64 || (first > 0 && snk < 64)) {
#pragma unroll
                    for (int q = 0; q < 2; ++q) {
                        const uint32_t see = below(last - 32 * q) & (~below(first - 32 * q) | below(snk - 32 * q));
#pragma unroll
                        for (int c = 0; c < 32; ++c)
                            if (!(see & (1u << c))) s[q][c] = __float_as_uint(-INFINITY);
                    }
                }

                float mx0 = -INFINITY, mx1 = -INFINITY;
#pragma unroll
                for (int c = 0; c < 32; c += 2) {
                    mx0 = fmax3_nan(mx0, __uint_as_float(s[0][c]), __uint_as_float(s[0][c + 1]));
                    mx1 = fmax3_nan(mx1, __uint_as_float(s[1][c]), __uint_as_float(s[1][c + 1]));
                }
                float mx = fmax_nan(mx0, mx1);
                mx = fmax_nan(mx, __shfl_xor_sync(0xffffffffu, mx, 16));
                const float m_new = mx * p.scale_log2;
                // Lazy rescale: keep the old maximum unless the tile's exceeds it by more than
                // 8 (log2 units). A row that has seen nothing yet refers to 0, so that its
                // masked scores give 2^-inf and not NaN. A NaN score makes the row's maximum NaN and
                // so, through alpha, its sum, whichever columns the FMA-pipe exponential takes (it
                // has no NaN of its own); the comparison is written for that.
                float alpha = 1.f;
                const bool need = !(m_new <= m_use + 8.0f);
                if (need) {
                    alpha = fast_exp2(m_use - m_new);
                    m_use = m_new;
                }
                const float neg_m = m_use == -INFINITY ? 0.f : kShift - m_use;

                uint32_t pk[2][16];
                const uint64_t negm_2 = f2_pack(neg_m, neg_m);
                uint64_t sum_a = f2_pack(0.f, 0.f), sum_b = f2_pack(0.f, 0.f);
#pragma unroll
                for (int q = 0; q < 2; ++q) {
#pragma unroll
                    for (int c = 0; c < 16; ++c) {
                        const uint64_t x2 =
                            f2_fma(f2_pack(__uint_as_float(s[q][2 * c]), __uint_as_float(s[q][2 * c + 1])), sl2_2, negm_2);
                        uint64_t p2;
                        // At d = 64 one pair of eight takes the FMA pipe, as in the dense kernel; at
                        // d = 128 MUFU has headroom.
                        if (D == 64 && ((q * 16 + c) & 7) == 0) {
                            p2 = exp2_poly_x2<true>(x2);
                        } else {
                            float x0, x1;
                            f2_unpack(x2, x0, x1);
                            p2 = f2_pack(fast_exp2(x0), fast_exp2(x1));
                        }
                        if (c & 1)
                            sum_b = f2_add(sum_b, p2);
                        else
                            sum_a = f2_add(sum_a, p2);
                        float p0, p1;
                        f2_unpack(p2, p0, p1);
                        pk[q][c] = kF16 ? pack_f16x2(p0, p1) : pack_bf16x2(p0, p1);
                    }
                }
                {
                    float a0, a1, b0, b1;
                    f2_unpack(sum_a, a0, a1);
                    f2_unpack(sum_b, b0, b1);
                    l_half = l_half * alpha + ((a0 + a1) + (b0 + b1));
                }

                // PV_t of the previous step has read P_t and O_t is final. At d = 128 that held
                // before S_t was issued.
                if (C::kSepP && g > 0) {
                    if (!(ok = warp_wait(bar_pv, (g - 1) & 1u, ctl, kSiteSoftPV))) break;
                    tc_fence_after();
                }
                if (s_i > 0 && __any_sync(0xffffffffu, need)) {
#pragma unroll 1
                    for (int part = 0; part < D / 64; ++part) {
                        uint32_t o[32];
                        tmem_ld16x32bx2_x32<D / 2>(tO + 32 * part, o);
                        tmem_wait_ld();
#pragma unroll
                        for (int c = 0; c < 32; ++c) o[c] = __float_as_uint(__uint_as_float(o[c]) * alpha);
                        tmem_st16x32bx2_x32<D / 2>(tO + 32 * part, o);
                    }
                }
                tmem_st16x32bx2_x16<32>(tP, pk[0]);
                tmem_st16x32bx2_x16<32>(tP + 16, pk[1]);
                tmem_wait_st();
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(bar_p);
            }
            if (!ok) break;

            // ---------------------------------------------------- epilogue of this item
            if (steps > 0) {
                if (!(ok = warp_wait(bar_pv, (g - 1) & 1u, ctl, kSiteSoftPV))) break;
                tc_fence_after();
            }
            float l_sum = l_half + __shfl_xor_sync(0xffffffffu, l_half, 16);
            // A score of +inf stays the maximum, and its weight is 2^(inf - inf): the row is NaN.
            if (m_use == INFINITY) l_sum = NAN;
            const bool empty = m_use == -INFINITY && l_sum == l_sum;  // a row of NaN scores is not empty
            const float inv = empty ? 0.f : 1.f / l_sum;
            const float lse2 = empty ? -INFINITY : m_use - kShift + __log2f(l_sum);
            // Decoded afresh: kept from above, it would take registers from the steps.
            Item it;
            int item_again = item;
            asm volatile("" : "+r"(item_again));
            decode<kPartial>(p, item_again, it);
            size_t idx;
            bool row_ok;
            if constexpr (kPartial) {
                const int sb = p.seqs_per_tile ? row / p.q_rows : 0;
                const int b = pick(it.b, t) + sb;
                const int r = p.seqs_per_tile ? row - sb * p.q_rows : pick(it.row0, t) + row;
                row_ok = pick(it.hi, t) > 0 && b < p.batch && r < p.q_rows && (!p.seqs_per_tile || sb < p.seqs_per_tile);
                idx = (size_t)it.split * p.rows + ((size_t)b * p.hkv + it.kvh) * p.q_rows + r;
            } else {
                const int q_row = pick(it.row0, t) + row;
                row_ok = q_row < p.n_q;
                idx = ((size_t)pick(it.b, t) * p.hq + pick(it.head, t)) * p.n_q + q_row;
            }
#pragma unroll 1
            for (int part = 0; part < D / 64; ++part) {
                uint32_t o[32];
                tmem_ld16x32bx2_x32<D / 2>(tO + 32 * part, o);  // without steps: anything, and not used
                tmem_wait_ld();
                if (empty) {
#pragma unroll
                    for (int c = 0; c < 32; ++c) o[c] = 0u;
                }
                if (row_ok) {
                    const size_t at = idx * D + h * (D / 2) + part * 32;
                    if constexpr (kPartial) {
                        float* dst = reinterpret_cast<float*>(p.out) + at;
#pragma unroll
                        for (int c = 0; c < 4; ++c) {
                            uint32_t w[8];
#pragma unroll
                            for (int e = 0; e < 8; ++e) w[e] = __float_as_uint(__uint_as_float(o[8 * c + e]) * inv);
                            st_global_v8(dst + 8 * c, w);
                        }
                    } else {
                        uint16_t* dst = reinterpret_cast<uint16_t*>(p.out) + at;
#pragma unroll
                        for (int c = 0; c < 2; ++c) {
                            uint32_t w[8];
#pragma unroll
                            for (int e = 0; e < 8; ++e) {
                                const float a = __uint_as_float(o[16 * c + 2 * e]) * inv;
                                const float b = __uint_as_float(o[16 * c + 2 * e + 1]) * inv;
                                w[e] = kF16 ? pack_f16x2(a, b) : pack_bf16x2(a, b);
                            }
                            st_global_v8(dst + 16 * c, w);
                        }
                    }
                }
            }
            // The next item's first PV overwrites O_t: the loads above have completed before
            // this warp arrives on p_full again.
            if (row_ok && h == 0 && p.lse) p.lse[idx] = kPartial ? lse2 : lse2 * 0.69314718055994531f;
        }
    } else if (warp == kProducerWarp) {
        // ------------------------------------------------------------ TMA producer
        const bool leader = elect_one();
        const uint32_t q_smem0 = smem_addr(smem + C::kOffQ);
        const uint32_t k_smem0 = smem_addr(smem + C::kOffK), v_smem0 = smem_addr(smem + C::kOffV);
        const uint32_t q_bytes =
            (uint32_t)C::kChunks * (kPartial && p.seqs_per_tile ? p.seqs_per_tile * p.q_rows * 128 : C::kChunkBytes);
        int last_k = -1, last_v = -1, last_q = -1;
        int c = 0, st = 0, n_it = 0;
        uint32_t par = 1u;
        bool ok = true;
        for (int item = blockIdx.x; item < p.items && ok; item += gridDim.x) {
            Item it;
            decode<kPartial>(p, item, it);
            if (it.steps == 0) continue;
            const int qb = n_it % C::kQBufs;
            if (!(ok = warp_wait(smem_addr(&bars->q_empty[qb]), (uint32_t)(n_it / C::kQBufs & 1) ^ 1u, ctl, kSiteProdQ)))
                break;
            if (leader) {
                for (int t = 0; t < 2; ++t) {
                    const uint32_t qf = smem_addr(&bars->q_full[qb][t]);
                    mbar_arrive_expect_tx(qf, q_bytes);
                    for (int ch = 0; ch < C::kChunks; ++ch)
                        tma_load_4d(q_smem0 + (qb * 2 + t) * C::kTile + ch * C::kChunkBytes, &tmQ, qf, ch * 64,
                                    it.row0[t], kPartial ? it.b[t] : it.head[t], kPartial ? it.kvh : it.b[t]);
                }
            }
            last_q = n_it++;
            __syncwarp();
            for (int s_i = 0; s_i < it.steps; ++s_i, ++c) {
                const int j = step_tile(it, s_i);
                const uint32_t kf = smem_addr(&bars->k_full[st]), vf = smem_addr(&bars->v_full[st]);
                if (!(ok = warp_wait(smem_addr(&bars->k_empty[st]), par, ctl, kSiteProdK))) break;
                if (leader) {
                    mbar_arrive_expect_tx(kf, C::kTile);
                    for (int ch = 0; ch < C::kChunks; ++ch)
                        tma_load_4d(k_smem0 + st * C::kTile + ch * C::kChunkBytes, &tmK, kf, ch * 64, j * 128, it.kvh,
                                    it.kvb);
                }
                last_k = c;
                __syncwarp();
                if (!(ok = warp_wait(smem_addr(&bars->v_empty[st]), par, ctl, kSiteProdV))) break;
                if (leader) {
                    mbar_arrive_expect_tx(vf, C::kTile);
                    for (int ch = 0; ch < C::kChunks; ++ch)
                        tma_load_4d(v_smem0 + st * C::kTile + ch * C::kChunkBytes, &tmV, vf, ch * 64, j * 128, it.kvh,
                                    it.kvb);
                }
                last_v = c;
                __syncwarp();
                if (++st == C::kStages) {
                    st = 0;
                    par ^= 1u;
                }
            }
        }
        if (*ctl.abort_flag) {
            // Let copies still in flight land before the CTA's shared memory is released.
            int never = 0;
            const WaitCtl drain{&never, nullptr, ctl.limit_ns};
            for (int s = 0; s < C::kStages; ++s) {
                if (last_k - s >= 0)
                    mbar_wait(smem_addr(&bars->k_full[(last_k - s) % C::kStages]),
                              (uint32_t)((last_k - s) / C::kStages) & 1u, drain, 0);
                if (last_v - s >= 0)
                    mbar_wait(smem_addr(&bars->v_full[(last_v - s) % C::kStages]),
                              (uint32_t)((last_v - s) / C::kStages) & 1u, drain, 0);
            }
            for (int s = 0; s < C::kQBufs; ++s)
                if (last_q - s >= 0)
                    for (int t = 0; t < 2; ++t)
                        mbar_wait(smem_addr(&bars->q_full[(last_q - s) % C::kQBufs][t]),
                                  (uint32_t)((last_q - s) / C::kQBufs) & 1u, drain, 0);
        }
        __syncwarp();
    } else {
        // ------------------------------------------------------------ MMA issuers
        constexpr uint32_t kFmt = kF16 ? ~((1u << 7) | (1u << 10)) : ~0u;  // A and B format bits: 0 = fp16, 1 = bf16
        constexpr uint32_t kIdescS = idesc_bf16_f32(128, 128, 0) & kFmt;
        constexpr uint32_t kIdescSh = idesc_bf16_f32(128, 64, 0) & kFmt;
        constexpr uint32_t kIdescSn = idesc_bf16_f32(128, 32, 0) & kFmt;
        constexpr uint32_t kHalfRowsLo = (64 * 128) >> 4;  // K rows 64.. inside a chunk
        constexpr uint32_t kIdescO = idesc_bf16_f32(128, 64, 1) & kFmt;
        constexpr uint32_t kChunkLo = C::kChunkBytes >> 4;
        constexpr uint32_t kTileLo = C::kTile >> 4;
        const uint32_t on = elect_one() ? 1u : 0u;
        const uint64_t desc_base = smem_desc_sw128(smem_addr(smem), 16, 1024);
        const uint32_t desc_hi = (uint32_t)(desc_base >> 32);
        const uint32_t lo0 = (uint32_t)desc_base;
        const uint32_t v_lo0 = lo0 + (C::kOffV >> 4);
        const bool is_pv = warp == kPVWarp;
        const int ts = warp == kSWarp ? 0 : 1;  // S issuers: their tile
        uint32_t g[2] = {0, 0};                 // steps of tile t so far
        uint32_t st = 0, par = 0;
        int n_it = 0;
        bool ok = true;
        for (int item = blockIdx.x; item < p.items && ok; item += gridDim.x) {
            Item it;
            decode<kPartial>(p, item, it);
            if (it.steps == 0) continue;
            const int qb = n_it % C::kQBufs;
            const uint32_t q_par = (uint32_t)(n_it / C::kQBufs) & 1u;
            ++n_it;
            bool first[2] = {true, true};
            for (int s_i = 0; s_i < it.steps; ++s_i) {
                const int j = step_tile(it, s_i);
                if (!is_pv) {
                    if (!(ok = warp_wait(smem_addr(&bars->k_full[st]), par, ctl, kSiteMmaK))) break;
                    // An idle tile's query load, too, must land before its buffer is reused.
                    if (s_i == 0 && !(ok = warp_wait(smem_addr(&bars->q_full[qb][ts]), q_par, ctl, kSiteMmaQ + ts))) break;
                    if (sees(p, it, ts, j)) {
                        const uint32_t k_lo = lo0 + (C::kOffK >> 4) + st * kTileLo;
                        const uint32_t q_lo = lo0 + (C::kOffQ >> 4) + (uint32_t)(qb * 2 + ts) * kTileLo;
                        const uint32_t d = tmem + ts * 128;
                        const bool narrow = kNarrow && j < pick(it.lo, ts);
                        if (g[0] > 0 && !(ok = warp_wait(smem_addr(&bars->s_empty[ts]), (g[0] - 1) & 1u, ctl, kSiteMmaK + 3 + ts)))
                            break;
                        tc_fence_after();
                        if (narrow) {  // keys 0..31 alone
                            if (!C::kSepP && g[0] > 0 &&
                                !(ok = warp_wait(smem_addr(&bars->pv_done[ts]), (g[0] - 1) & 1u, ctl, kSiteMmaK + 1 + ts)))
                                break;
                            tc_fence_after();
#pragma unroll
                            for (int kk = 0; kk < D / 16; ++kk) {
                                const uint32_t off = (uint32_t)(kk >> 2) * kChunkLo + (uint32_t)(kk & 3) * 2;
                                umma_ss_on(on, d, q_lo + off, k_lo + off, desc_hi, kIdescSn, kk > 0);
                            }
                        } else if constexpr (C::kSepP) {
#pragma unroll
                            for (int kk = 0; kk < D / 16; ++kk)
                                umma_ss_on(on, d, q_lo + kk * 2, k_lo + kk * 2, desc_hi, kIdescS, kk > 0);
                        } else {
                            // Keys 64..127 as soon as S_t has been loaded; keys 0..63, where P_t lives,
                            // after PV_t of the previous step has read P_t.
#pragma unroll
                            for (int kk = 0; kk < D / 16; ++kk) {
                                const uint32_t off = (uint32_t)(kk >> 2) * kChunkLo + (uint32_t)(kk & 3) * 2;
                                umma_ss_on(on, d + 64, q_lo + off, k_lo + off + kHalfRowsLo, desc_hi, kIdescSh, kk > 0);
                            }
                            if (g[0] > 0 &&
                                !(ok = warp_wait(smem_addr(&bars->pv_done[ts]), (g[0] - 1) & 1u, ctl, kSiteMmaK + 1 + ts)))
                                break;
                            tc_fence_after();
#pragma unroll
                            for (int kk = 0; kk < D / 16; ++kk) {
                                const uint32_t off = (uint32_t)(kk >> 2) * kChunkLo + (uint32_t)(kk & 3) * 2;
                                umma_ss_on(on, d, q_lo + off, k_lo + off, desc_hi, kIdescSh, kk > 0);
                            }
                        }
                        umma_commit_on(on, smem_addr(&bars->s_full[ts]));
                        ++g[0];
                    }
                    umma_commit_on(on, smem_addr(&bars->k_empty[st]));
                    if (s_i == it.steps - 1) umma_commit_on(on, smem_addr(&bars->q_empty[qb]));
                    __syncwarp();
                } else {
                    if (!(ok = warp_wait(smem_addr(&bars->v_full[st]), par, ctl, kSiteMmaV))) break;
                    const uint32_t v_lo = v_lo0 + st * kTileLo;
#pragma unroll
                    for (int t = 0; t < 2; ++t) {
                        if (!sees(p, it, t, j)) continue;
                        if (!(ok = warp_wait(smem_addr(&bars->p_full[t]), g[t] & 1u, ctl, kSiteMmaV + 1 + t))) break;
                        tc_fence_after();
                        const uint32_t rest = kNarrow && j < it.lo[t] ? 0u : on;  // past key 31
#pragma unroll
                        for (int kk = 0; kk < 8; ++kk)  // 16 keys: 8 TMEM columns of P, 16 x 128 bytes of V
#pragma unroll
                            for (int ch = 0; ch < C::kChunks; ++ch)
                                umma_ts_on(kk < 2 ? on : rest, tmem + C::kColO + t * D + ch * 64, tmem + C::kColP + t * C::kStepP + kk * 8,
                                           v_lo + ch * kChunkLo + kk * 128, desc_hi, kIdescO, !first[t] || kk > 0);
                        umma_commit_on(on, smem_addr(&bars->pv_done[t]));
                        first[t] = false;
                        ++g[t];
                    }
                    if (!ok) break;
                    umma_commit_on(on, smem_addr(&bars->v_empty[st]));
                    __syncwarp();
                }
                if (++st == C::kStages) {
                    st = 0;
                    par ^= 1u;
                }
            }
        }
        // Drain: every MMA this warp issued has finished before TMEM is released.
        const uint32_t drain_bar = smem_addr(&bars->drain[warp - kSWarp]);
        umma_commit_on(on, drain_bar);
        __syncwarp();
        int never = 0;
        const WaitCtl drain{&never, nullptr, ctl.limit_ns};
        mbar_wait(drain_bar, 0u, drain, 0);
        __syncwarp();
    }

    tc_fence_before();
    __syncthreads();
    if (warp == kSWarp) {
        tc_fence_after();
        tmem_dealloc(tmem, kTmemCols);
    }
}

}  // namespace win
