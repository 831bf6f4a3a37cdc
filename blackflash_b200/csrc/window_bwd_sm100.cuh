// Backward of the sliding-window attention for sm_100a (included by window_sm100.cu inside
// namespace bfk, after the forward). With P = exp(scale Q K^T - lse) over the visible pairs
// and D_i = sum_c dO_ic O_ic,
//
//   dS = P o (dO V^T - D),  dV = P^T dO,  dK = scale dS^T Q,  dQ = scale dS K,
//
// dK and dV summed over the query heads of a KV head.
//
// Two passes instead of one: dK / dV per KV tile and dQ per query tile, each recomputing S
// and dO V^T. That is seven products instead of five, but nothing is added through global
// memory: no fp32 accumulator of dQ is cleared, added to and read back (with a window each
// tile meets only a few others, so that traffic would rival the products), no atomics, and
// the result does not depend on the order of the blocks.
//
// Both passes are one kernel. A work item keeps two stationary 128-row tiles X0, X1 and
// streams pairs of 64-row tiles Y0, Y1 past them:
//                    X0  X1   Y0  Y1    S = X0 Y0^T   dP = X1 Y1^T   accumulators
//   dK/dV (kDQ=0)    K   V    Q   dO    (S^T)         (dP^T)         dV += P^T Y1, dK += dS^T Y0
//   dQ    (kDQ=1)    Q   dO   K   V                                  dQ += dS Y0
// D. Both passes read it from an array that the prep kernel fills from O. O is rounded to
// bf16, and for a row that sees few keys that error is not small against dP - D, of which D
// is then a large part (one key: dP - D is 0). So a query tile with such a row (the first of a
// sequence, or every one of a short window) walks its KV tiles twice in the dQ pass: first it
// sums P dP and P in fp32, D = sum P dP / sum P, which it also leaves in the array for the
// dK/dV pass; then it accumulates.
// Roles: two groups of eight elementwise warps (two threads per row), which take the steps in
// turn: a step is a chain of TMEM loads, exponentials and stores that one group alone leaves
// mostly waiting, so the other one's chain runs under it; a TMA producer; one issuer each of S,
// dP and the accumulations (an MMA takes about 60 cycles to issue here, so one warp for S and
// dP was itself the limit). Blocks are persistent, so an item's tail overlaps the next one's
// first products.
// TMEM (512 columns): four 64-column buffers, the accumulators from 256 on. Everything of a
// step happens in one buffer: S is computed there and loaded; dP is computed over it while the
// exponentials run; P and dS, as bf16 the A operands of the accumulations, go over dP. With two
// buffers a group, no step waits for the accumulations of the step before (with S and dP
// buffers apart, one each a group, it did: 1970 cycles a step against the tensor core's 1020).
// P stays fp32 until it is multiplied by dP - D, so that dS is rounded once. In the dK/dV pass
// lse and D go by column, the same for all rows: read from shared memory by every thread they
// took a third of its bandwidth. There the tensor core subtracts them instead: each query has 16
// bytes more, -lse / scale and -D in three bf16 terms each (24 bits), which one more K = 16
// product adds to S and to dP against stationary rows of ones and zeros. 64-row streamed
// tiles leave that room, and 32 columns a thread fit the 104 registers that sixteen
// elementwise warps can have; the price is that S and dP, 64 wide, are bound by reading their
// stationary operand from shared memory (48 cycles an MMA instead of 32).
namespace winb {

using win::kTmemCols;

constexpr int kThreads = 20 * 32;
constexpr int kGroupWarps = 8, kEwWarps = 2 * kGroupWarps;
constexpr int kProdWarp = 16;
constexpr int kFrontWarp = 17;  // issues S (and owns the TMEM allocation); 18 dP; 19 the accumulations
constexpr int kEwRegs = 104, kOtherRegs = 64;  // launch budget 640 x 96
static_assert(kEwWarps * 32 * kEwRegs + 128 * kOtherRegs <= kThreads * 96, "register split exceeds the launch budget");
constexpr int NT = 64;       // rows of a streamed tile
constexpr int NC = NT / 2;   // of them (S columns) a thread's
constexpr int kFewKeys = 128;  // D from fp32 sums for tiles with a row that sees at most so many
constexpr int kBufs = 4;     // S / dP / P, dS buffers; step n uses buffer n % 4
constexpr int kColAcc = kBufs * NT;

template <int D, bool kDQ>
struct Cfg {
    static constexpr int kChunks = D / 64;
    static constexpr int kXChunk = 128 * 128, kXTile = kChunks * kXChunk;
    static constexpr int kYChunk = NT * 128, kYTile = kChunks * kYChunk;
    static constexpr int kStages = D == 128 ? 4 : 6;
    static constexpr int kVec = kDQ ? 0 : NT * 16;  // dK/dV: a tile's rows of Params::aug
    static constexpr int kOffX = 0;
    static constexpr int kOffY = kOffX + 2 * kXTile;              // [kStages][Y0, Y1]
    static constexpr int kOffVec = kOffY + kStages * 2 * kYTile;  // [kStages]
    // dK/dV: 128 rows of 16 bytes with ones at -D's terms, 128 with ones at -lse's, 128 of
    // zeros. dQ: [2][2 groups][128] {sum P, sum P dP}.
    static constexpr int kOffOnes = kOffVec + kStages * kVec;
    static constexpr int kOffSum = kOffOnes;
    static constexpr int kOffBar = kOffOnes + (kDQ ? 4096 : 3 * 2048);
    static constexpr int kAccs = kDQ ? 1 : 2;
    static_assert(kColAcc + kAccs * D <= kTmemCols, "TMEM columns");
};

template <int D, bool kDQ>
struct Bars {
    uint64_t x_full, x_empty;
    uint64_t y_full[Cfg<D, kDQ>::kStages], y_empty[Cfg<D, kDQ>::kStages];
    uint64_t s_full[kBufs], s_read[kBufs];    // S computed; loaded by the group
    uint64_t dp_full[kBufs], p_ready[kBufs];  // dP computed; P, dS written
    uint64_t buf_free[kBufs];                 // the accumulations have read P, dS
    uint64_t acc_full, acc_free;
    uint64_t sums;  // dQ, two sweeps: every warp's sums are in shared memory
    uint64_t drain[3];
    uint32_t tmem_base;
    int abort_flag;
};

template <int D, bool kDQ>
constexpr int smem_bytes() {
    return Cfg<D, kDQ>::kOffBar + (int)sizeof(Bars<D, kDQ>) + 1024;
}
static_assert(smem_bytes<64, false>() <= 227 * 1024 && smem_bytes<128, false>() <= 227 * 1024 &&
                  smem_bytes<64, true>() <= 227 * 1024 && smem_bytes<128, true>() <= 227 * 1024,
              "shared memory");

enum : unsigned {
    kSiteProdX = 0x800,
    kSiteProdY = 0x801,
    kSiteFrontX = 0x810,
    kSiteFrontY = 0x811,
    kSiteFrontS = 0x812,
    kSiteFrontDP = 0x813,
    kSiteAccP = 0x820,
    kSiteAccFree = 0x821,
    kSiteEwS = 0x830,
    kSiteEwDP = 0x831,
    kSiteEwAcc = 0x832,
    kSiteEwSums = 0x833,
};

struct Params {
    int items;
    // dK/dV: blocks take their items at places blockIdx, blockIdx + gridDim, .. of a list that has
    // `late_rows` rows, from place late_from on, with holes for its first late_blocks blocks.
    int places, late_from, late_rows, late_blocks;
    int batch, hq, hkv, group;
    int n_q, n_kv, n_pad;    // n_pad: n_q rounded up to 128, row stride of nlse2 / nd
    int nk, ns;              // KV tiles; of them tiles that hold sinks
    int window, sinks;       // clamped to n_kv
    int q_tiles;             // 128-row query tiles (dQ)
    int splits_s, splits_n;  // dK/dV: parts of a sink tile's and of another tile's queries
    float scale, scale_log2;
    const float* nlse2;      // [B Hq, n_pad] -lse log2(e); -inf past n_q and for rows that see nothing
    const float* nd;         // [B Hq, n_pad] -D
    uint4* aug;              // [B Hq, n_pad] eight bf16: -lse / scale in three terms, -D in three, 0, 0
    __nv_bfloat16 *dq, *dk, *dv;
    float* part;             // [slot][dV, dK][128][D] of the tiles with more than one part
    unsigned long long timeout_ns;
};

struct Item {
    int b, kvh, head;   // head: the query head (dQ)
    int tile;           // stationary 128-row tile
    int steps;          // dQ: of one sweep
    int lead;           // dQ: steps of a first sweep, which finds D and stores it in aug, or 0
    int i0, ni, s0;     // dK/dV: step s is query tile i0 + (s0 + s) % ni of head (s0 + s) / ni
    int n_sink, skip;   // dQ: step s is KV tile s, or s + skip past the sink tiles
    long long slot;     // dK/dV: part to write, -1: the gradient itself
};

// First query tile and number of query tiles (NT rows) that see KV tile j.
__device__ __forceinline__ void queries_of(const Params& p, int j, int& i0, int& ni) {
    const int off = p.n_kv - p.n_q;
    const int last_key = min(j * 128 + 127, p.n_kv - 1);
    const int lo = max(0, j * 128 - off);
    const int hi = j < p.ns ? p.n_q : min(p.n_q, last_key + p.window - off);
    i0 = lo / NT;
    ni = hi > lo ? (hi + NT - 1) / NT - i0 : 0;
}

// x in three bf16 terms: hi + mid + lo is x to 24 bits.
__device__ __forceinline__ void split3(float x, uint32_t& hi, uint32_t& mid, uint32_t& lo) {
    hi = pack_bf16x2(x, 0.f) & 0xffffu;
    x -= __uint_as_float(hi << 16);
    mid = pack_bf16x2(x, 0.f) & 0xffffu;
    x -= __uint_as_float(mid << 16);
    lo = pack_bf16x2(x, 0.f) & 0xffffu;
}

// The item at a place of the list; at a hole or past the last item p.items.
template <bool kDQ>
__device__ __forceinline__ int item_at(const Params& p, int place) {
    if (kDQ || place < p.late_from) return place;
    const int row = (place - p.late_from) / (int)gridDim.x, gap = p.late_blocks;
    if (row >= p.late_rows) return min(place - p.late_rows * gap, p.items);
    const int item = place - (row + 1) * gap;  // of the blocks from `gap` on
    return (int)blockIdx.x < gap ? p.items : min(item, p.items);
}

template <int D, bool kDQ>
__device__ __forceinline__ void decode(const Params& p, int item, Item& it) {
    if constexpr (kDQ) {
        // Late rows see the most keys: first. Heads of a group are neighbours and share K/V in L2.
        const int units = p.batch * p.hq;
        const int unit = item % units;
        it.tile = p.q_tiles - 1 - item / units;
        it.b = unit / p.hq;
        it.head = unit % p.hq;
        it.kvh = it.head / p.group;
        const int off = p.n_kv - p.n_q;
        const int p_first = it.tile * 128 + off, p_last = min(it.tile * 128 + 128, p.n_q) - 1 + off;
        const int lo = max(0, p_first - p.window + 1) / NT;
        const int hi = p_last >= 0 ? p_last / NT + 1 : 0;
        it.n_sink = min((p.sinks + NT - 1) / NT, lo);
        it.skip = lo - it.n_sink;
        it.steps = hi > 0 ? hi - it.skip : 0;
        // The tile's first row sees min(p_first + 1, window + sinks) keys, the fewest of its rows.
        it.lead = p_first < kFewKeys || p.window <= kFewKeys - p.sinks ? it.steps : 0;
        it.slot = -1;
    } else {
        it.lead = 0;
        // Sink tiles first, in parts (all later queries see them); early keys are seen most.
        const int units = p.batch * p.hkv;
        const int unit = item % units;
        int idx = item / units;
        it.b = unit / p.hkv;
        it.kvh = unit % p.hkv;
        int part, splits;
        const int sink_items = p.ns * p.splits_s;
        if (idx < sink_items) {
            splits = p.splits_s;
            it.tile = idx / splits;
            part = idx % splits;
            it.slot = splits > 1 ? ((long long)unit * p.ns + it.tile) * splits + part : -1;
        } else {
            idx -= sink_items;
            splits = p.splits_n;
            it.tile = p.ns + idx / splits;
            part = idx % splits;
            const long long base = p.splits_s > 1 ? (long long)units * sink_items : 0;
            it.slot = splits > 1 ? base + ((long long)unit * (p.nk - p.ns) + it.tile - p.ns) * splits + part : -1;
        }
        queries_of(p, it.tile, it.i0, it.ni);
        const long long len = (long long)it.ni * p.group;
        it.s0 = (int)(len * part / splits);
        it.steps = (int)(len * (part + 1) / splits) - it.s0;
    }
}

template <int D, bool kDQ>
__global__ void __launch_bounds__(kThreads, 1)
    window_bwd_kernel(const __grid_constant__ CUtensorMap tmX0, const __grid_constant__ CUtensorMap tmX1,
                      const __grid_constant__ CUtensorMap tmY0, const __grid_constant__ CUtensorMap tmY1, const Params p) {
    using C = Cfg<D, kDQ>;
    extern __shared__ uint8_t smem_raw[];
    uint8_t* smem = align1024(smem_raw);
    Bars<D, kDQ>* bars = reinterpret_cast<Bars<D, kDQ>*>(smem + C::kOffBar);
    const int warp = __shfl_sync(0xffffffffu, (int)(threadIdx.x >> 5), 0);  // known to be uniform
    const int lane = threadIdx.x & 31;

    if (threadIdx.x == 0) {
        mbar_init(smem_addr(&bars->x_full), 1);
        mbar_init(smem_addr(&bars->x_empty), 2);  // S and dP each
        for (int s = 0; s < C::kStages; ++s) {
            mbar_init(smem_addr(&bars->y_full[s]), 1);
            mbar_init(smem_addr(&bars->y_empty[s]), 1);
        }
        for (int b = 0; b < kBufs; ++b) {
            mbar_init(smem_addr(&bars->s_full[b]), 1);
            mbar_init(smem_addr(&bars->s_read[b]), kGroupWarps);  // one arrival per elementwise warp of the group
            mbar_init(smem_addr(&bars->dp_full[b]), 1);
            mbar_init(smem_addr(&bars->p_ready[b]), kGroupWarps);
            mbar_init(smem_addr(&bars->buf_free[b]), 1);
        }
        for (int r = 0; r < 3; ++r) mbar_init(smem_addr(&bars->drain[r]), 1);
        mbar_init(smem_addr(&bars->acc_full), 1);
        mbar_init(smem_addr(&bars->acc_free), kEwWarps);
        mbar_init(smem_addr(&bars->sums), kEwWarps);
        bars->abort_flag = 0;
        fence_barrier_init();
    }
    if constexpr (!kDQ) {
        if (threadIdx.x < 384) {
            const uint32_t one = 0x3f80u;  // bf16
            uint4 v = make_uint4(0, 0, 0, 0);
            if (threadIdx.x < 128)
                v = make_uint4(0, one << 16, one | (one << 16), 0);
            else if (threadIdx.x < 256)
                v = make_uint4(one | (one << 16), one, 0, 0);
            *reinterpret_cast<uint4*>(smem + C::kOffOnes + threadIdx.x * 16) = v;
        }
        fence_proxy_async_smem();
    }
    if (warp == kProdWarp && lane == 0) {
        tma_prefetch_desc(&tmX0);
        tma_prefetch_desc(&tmX1);
        tma_prefetch_desc(&tmY0);
        tma_prefetch_desc(&tmY1);
    }
    if (warp == kFrontWarp) {
        tmem_alloc(smem_addr(&bars->tmem_base), kTmemCols);
        tmem_relinquish();
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = bars->tmem_base;
    const WaitCtl ctl{&bars->abort_flag, &g_wait_status, p.timeout_ns};
    griddep_launch_dependents();
    griddep_wait();  // nothing above touches global data

    if (warp < kEwWarps)
        regs_inc<kEwRegs>();
    else
        regs_dec<kOtherRegs>();

    if (warp < kEwWarps) {
        // ------------------------------------------------------------ elementwise
        const int grp = warp >> 3;  // takes the steps n with n % 2 == grp
        const int quarter = warp & 3;
        const int sub = (warp >> 2) & 1;
        const int h = lane >> 4;                                // S columns NC h .. NC h + NC - 1
        const int row = quarter * 32 + sub * 16 + (lane & 15);  // row of the tile == TMEM lane
        const uint32_t tl = tmem + ((uint32_t)(quarter * 32 + sub * 16) << 16);
        const int off = p.n_kv - p.n_q;
        const uint64_t sl2_2 = f2_pack(p.scale_log2, p.scale_log2);
        uint32_t n0 = 0;  // steps of the items before
        int n_it = 0;     // items with steps so far
        int n_swept = 0;  // of them with a first sweep
        bool ok = true;
        // dQ: the next item is decoded, and its rows' -lse2 and -D requested, before the current
        // one's gradients are waited for (dK/dV has more steps an item and no registers for it).
        Item next;
        float next_l = 0.f, next_d = 0.f;  // dQ (padded rows have entries)
        auto fetch = [&](int item) {
            if (item >= p.items) return;
            decode<D, kDQ>(p, item, next);
            if constexpr (kDQ) {
                const size_t at = ((size_t)next.b * p.hq + next.head) * p.n_pad + next.tile * 128 + row;
                next_l = p.nlse2[at];
                next_d = next.lead > 0 ? 0.f : p.nd[at];
            }
        };
        if constexpr (kDQ) fetch(blockIdx.x);
        for (int place = blockIdx.x; place < p.places && ok; place += gridDim.x) {
            const int item = item_at<kDQ>(p, place);
            if (item >= p.items) continue;
            if constexpr (!kDQ) fetch(item);
            const Item it = next;
            const int xrow = it.tile * 128 + row;
            const int lead = it.lead;
            uint64_t nl2 = f2_pack(next_l, next_l), nd2 = f2_pack(next_d, next_d);
            int q_tile = 0;  // dK/dV: the next step's query tile, from i0 on
            // One step; in the first sweep (measure) it only adds up P and P dP.
            float sum_p = 0.f, sum_pdp = 0.f;
            auto step = [&](int s_i, uint32_t n, bool measure) -> bool {
                const uint32_t buf = n & (kBufs - 1), par = (n / kBufs) & 1u;
                const uint32_t tB = tl + buf * NT;
                // Visible: column c with c < last and (c >= first or c < snk).
                int first, last, snk;
                if constexpr (kDQ) {
                    const int c0 = (s_i < it.n_sink ? s_i : s_i + it.skip) * NT + h * NC;
                    last = xrow + off + 1 - c0;
                    first = xrow + off + 1 - p.window - c0;
                    snk = p.sinks - c0;
                } else {
                    const int q0 = (it.i0 + q_tile) * NT + h * NC;
                    first = xrow - off - q0;
                    last = xrow < p.sinks ? NC : first + p.window;
                    snk = 0;
                }
                if (!warp_wait(smem_addr(&bars->s_full[buf]), par, ctl, kSiteEwS)) return false;
                tc_fence_after();
                float pr[NC];
                {
                    uint32_t s[NC];
                    tmem_ld16x32bx2_x32<NC>(tB, s);
                    tmem_wait_ld();
                    tc_fence_before();
                    __syncwarp();
                    if (lane == 0) mbar_arrive(smem_addr(&bars->s_read[buf]));  // dP may be computed over it
#pragma unroll
                    for (int c = 0; c < NC; ++c) pr[c] = __uint_as_float(s[c]);
                }
                const bool edge = last < NC || (first > 0 && snk < NC);
                if (edge) {
                    const uint32_t see = win::below(last) & (~win::below(first) | win::below(snk));  // a bit per column
#pragma unroll
                    for (int c = 0; c < NC; ++c)
                        if (!(see & (1u << c))) pr[c] = -INFINITY;
                }
#pragma unroll
                for (int c = 0; c < NC; c += 2) {
                    float x0, x1;  // dK/dV: S has its -lse already, nl2 is 0
                    f2_unpack(f2_fma(f2_pack(pr[c], pr[c + 1]), sl2_2, nl2), x0, x1);
                    pr[c] = fast_exp2(x0);
                    pr[c + 1] = fast_exp2(x1);
                }
                // dS = P (dP - D)
                if (!warp_wait(smem_addr(&bars->dp_full[buf]), par, ctl, kSiteEwDP)) return false;
                tc_fence_after();
                uint32_t dp[NC];
                tmem_ld16x32bx2_x32<NC>(tB, dp);
                tmem_wait_ld();
                // P^T over the first half of the buffer (this thread: words NC h / 2 ..), dS^T over
                // the second; dQ needs dS alone.
                uint32_t pk[NC / 2];
                if constexpr (!kDQ) {
#pragma unroll
                    for (int c = 0; c < NC / 2; ++c) pk[c] = pack_bf16x2(pr[2 * c], pr[2 * c + 1]);
                    tmem_st16x32bx2_x16<NC / 2>(tB, pk);
                }
#pragma unroll
                for (int c = 0; c < NC; c += 2) {
                    uint64_t x = f2_pack(__uint_as_float(dp[c]), __uint_as_float(dp[c + 1]));
                    if constexpr (kDQ) x = f2_add(x, nd2);  // dK/dV: dP has its -D already
                    float x0, x1;
                    f2_unpack(f2_mul(x, f2_pack(pr[c], pr[c + 1])), x0, x1);
                    if (kDQ && measure) {  // D is 0 so far: x is P dP
                        if (pr[c] == 0.f) x0 = 0.f;
                        if (pr[c + 1] == 0.f) x1 = 0.f;
                        sum_p += pr[c] + pr[c + 1];
                        sum_pdp += x0 + x1;
                    }
                    pk[c / 2] = pack_bf16x2(x0, x1);
                }
                if (!measure) {
                    // dP of a masked pair may pass fp32, of large finite numbers, and 0 times it is
                    // NaN: a word of dS that has one is looked for in masked steps, and only then are
                    // the masked columns cleared. Looking takes 2.5 % of the backward at B=2 H=16
                    // N=4096 d=64 window 1024 (183 -> 187 us), 3.6 % at N=8192 window 256 (205 -> 213);
                    // clearing them in each masked step 7 and 16 %.
                    if (edge) {
                        uint32_t t0 = 0u, t1 = 0u;
#pragma unroll
                        for (int c = 0; c < NC / 2; c += 2) {
                            t0 = max_nan_bf16x2(t0, pk[c]);
                            t1 = max_nan_bf16x2(t1, pk[c + 1]);
                        }
                        t0 = max_nan_bf16x2(t0, t1);
                        if ((t0 & 0x7fffu) > 0x7f80u || (t0 & 0x7fff0000u) > 0x7f800000u) {
                            const uint32_t see = win::below(last) & (~win::below(first) | win::below(snk));
#pragma unroll
                            for (int c = 0; c < NC / 2; ++c)
                                pk[c] &= (see & (1u << (2 * c)) ? 0xffffu : 0u) | (see & (2u << (2 * c)) ? 0xffff0000u : 0u);
                        }
                    }
                    __syncwarp();
                    tmem_st16x32bx2_x16<NC / 2>(tB + (kDQ ? 0 : NT / 2), pk);
                    tmem_wait_st();
                }
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(smem_addr(&bars->p_ready[buf]));
                return true;
            };
            int s_all = (int)((n0 ^ (uint32_t)grp) & 1u);  // this group's first step of the item
            if constexpr (kDQ) {
                for (; s_all < lead && ok; s_all += 2) ok = step(s_all, n0 + s_all, true);
                if (!ok) break;
                if (lead > 0) {
                    // D from the four sums of the row: two column halves, two groups.
                    sum_p += __shfl_xor_sync(0xffffffffu, sum_p, 16);
                    sum_pdp += __shfl_xor_sync(0xffffffffu, sum_pdp, 16);
                    float2* sums = reinterpret_cast<float2*>(smem + C::kOffSum) + (n_swept & 1) * 256;
                    if (h == 0) sums[grp * 128 + row] = make_float2(sum_p, sum_pdp);
                    __syncwarp();
                    if (lane == 0) mbar_arrive(smem_addr(&bars->sums));
                    if (!(ok = warp_wait(smem_addr(&bars->sums), (uint32_t)n_swept & 1u, ctl, kSiteEwSums))) break;
                    ++n_swept;
                    const float2 x = sums[row], y = sums[128 + row];
                    const float tp = x.x + y.x, tpdp = x.y + y.y;
                    const float b = tp != 0.f ? -tpdp / tp : 0.f;  // a row that sees nothing has D = 0
                    nd2 = f2_pack(b, b);
                    if (grp == 0 && h == 0) {
                        uint32_t d0, d1, d2;
                        split3(b, d0, d1, d2);
                        uint32_t* a = reinterpret_cast<uint32_t*>(p.aug + ((size_t)it.b * p.hq + it.head) * p.n_pad + xrow);
                        reinterpret_cast<uint16_t*>(a)[3] = (uint16_t)d0;
                        a[2] = d1 | (d2 << 16);
                    }
                }
            }
            if constexpr (!kDQ) q_tile = it.ni > 0 ? (it.s0 + s_all) % it.ni : 0;
            for (; s_all < lead + it.steps && ok; s_all += 2) {
                ok = step(s_all - lead, n0 + s_all, false);
                if constexpr (!kDQ) {
                    q_tile += 2;
                    while (q_tile >= it.ni) q_tile -= it.ni;  // into the next head's tiles
                }
            }
            if (!ok) break;
            n0 += (uint32_t)(lead + it.steps);
            if constexpr (kDQ) fetch(item + gridDim.x);

            // ---------------------------------------------------- the item's gradients
            const bool any = it.steps > 0;
            if (any) {
                if (!(ok = warp_wait(smem_addr(&bars->acc_full), (uint32_t)n_it & 1u, ctl, kSiteEwAcc))) break;
                ++n_it;
                tc_fence_after();
            }
            // 32-column pieces of a thread: the groups take them in turn (dK/dV: 0 dV, 1 dK).
            constexpr int kPieces = C::kAccs * (D / 64);
#pragma unroll 1
            for (int i = grp ? (kPieces + 1) / 2 : 0; i < (grp ? kPieces : (kPieces + 1) / 2); ++i) {
                const int which = i / (D / 64), part = i % (D / 64);
                uint32_t o[32];
                tmem_ld16x32bx2_x32<D / 2>(tl + kColAcc + which * D + 32 * part, o);
                tmem_wait_ld();
                if (!any) {
#pragma unroll
                    for (int c = 0; c < 32; ++c) o[c] = 0u;
                }
                const int col = h * (D / 2) + 32 * part;
                const float f = kDQ || which ? p.scale : 1.f;
                if (it.slot >= 0) {
                    float* dst = p.part + ((it.slot * 2 + which) * 128 + row) * D + col;
#pragma unroll
                    for (int c = 0; c < 4; ++c) {
                        uint32_t w[8];
#pragma unroll
                        for (int e = 0; e < 8; ++e) w[e] = __float_as_uint(__uint_as_float(o[8 * c + e]) * f);
                        st_global_v8(dst + 8 * c, w);
                    }
                } else if (xrow < (kDQ ? p.n_q : p.n_kv)) {
                    __nv_bfloat16* dst = (kDQ ? p.dq + (((size_t)it.b * p.hq + it.head) * p.n_q + xrow) * D
                                              : (which ? p.dk : p.dv) + (((size_t)it.b * p.hkv + it.kvh) * p.n_kv + xrow) * D) +
                                         col;
#pragma unroll
                    for (int c = 0; c < 2; ++c) {
                        uint32_t w[8];
#pragma unroll
                        for (int e = 0; e < 8; ++e)
                            w[e] = pack_bf16x2(__uint_as_float(o[16 * c + 2 * e]) * f, __uint_as_float(o[16 * c + 2 * e + 1]) * f);
                        st_global_v8(dst + 16 * c, w);
                    }
                }
            }
            if (any) {  // the next item's first products may overwrite the accumulators
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(smem_addr(&bars->acc_free));
            }
        }
    } else if (warp == kProdWarp) {
        // ------------------------------------------------------------ TMA producer
        const bool leader = elect_one();
        const uint32_t xf = smem_addr(&bars->x_full);
        const uint32_t x0 = smem_addr(smem + C::kOffX), y0 = smem_addr(smem + C::kOffY), vec0 = smem_addr(smem + C::kOffVec);
        int n_it = 0, n = 0, st = 0;
        uint32_t par = 1u;
        bool ok = true;
        for (int place = blockIdx.x; place < p.places && ok; place += gridDim.x) {
            const int item = item_at<kDQ>(p, place);
            if (item >= p.items) continue;
            Item it;
            decode<D, kDQ>(p, item, it);
            if (it.steps == 0) continue;
            if (!(ok = warp_wait(smem_addr(&bars->x_empty), (uint32_t)(n_it & 1) ^ 1u, ctl, kSiteProdX))) break;
            if (leader) {
                mbar_arrive_expect_tx(xf, 2 * C::kXTile);
                const int head = kDQ ? it.head : it.kvh;
                for (int ch = 0; ch < C::kChunks; ++ch) {
                    tma_load_4d(x0 + ch * C::kXChunk, &tmX0, xf, ch * 64, it.tile * 128, head, it.b);
                    tma_load_4d(x0 + C::kXTile + ch * C::kXChunk, &tmX1, xf, ch * 64, it.tile * 128, head, it.b);
                }
            }
            ++n_it;
            __syncwarp();
            const int lead = it.lead;
            int g = 0, i = 0;  // dK/dV: head of the group and query tile of the next step
            if constexpr (!kDQ) {
                g = it.s0 / it.ni;
                i = it.s0 - g * it.ni;
            }
            for (int s_all = 0; s_all < lead + it.steps; ++s_all, ++n) {
                const int s_i = s_all < lead ? s_all : s_all - lead;
                const uint32_t f = smem_addr(&bars->y_full[st]);
                if (!(ok = warp_wait(smem_addr(&bars->y_empty[st]), par, ctl, kSiteProdY))) break;
                if (leader) {
                    int yrow, head;
                    if constexpr (kDQ) {
                        yrow = (s_i < it.n_sink ? s_i : s_i + it.skip) * NT;
                        head = it.kvh;
                    } else {
                        yrow = (it.i0 + i) * NT;
                        head = it.kvh * p.group + g;
                    }
                    mbar_arrive_expect_tx(f, 2 * C::kYTile + C::kVec);
                    const uint32_t y = y0 + (uint32_t)(st * 2 * C::kYTile);
                    for (int ch = 0; ch < C::kChunks; ++ch) {
                        tma_load_4d(y + ch * C::kYChunk, &tmY0, f, ch * 64, yrow, head, it.b);
                        tma_load_4d(y + C::kYTile + ch * C::kYChunk, &tmY1, f, ch * 64, yrow, head, it.b);
                    }
                    if constexpr (!kDQ) {
                        const size_t at = ((size_t)it.b * p.hq + head) * p.n_pad + yrow;
                        bulk_load(vec0 + st * C::kVec, p.aug + at, C::kVec, f);
                    }
                }
                __syncwarp();
                if (!kDQ && ++i == it.ni) {
                    i = 0;
                    ++g;
                }
                if (++st == C::kStages) {
                    st = 0;
                    par ^= 1u;
                }
            }
        }
        if (*ctl.abort_flag) {
            // Let copies still in flight land before the block's shared memory is released.
            int never = 0;
            const WaitCtl drain{&never, nullptr, ctl.limit_ns};
            if (n_it > 0) mbar_wait(xf, (uint32_t)(n_it - 1) & 1u, drain, 0);
            for (int s = 1; s <= C::kStages; ++s)
                if (n - s >= 0)
                    mbar_wait(smem_addr(&bars->y_full[(n - s) % C::kStages]), (uint32_t)((n - s) / C::kStages) & 1u, drain, 0);
        }
        __syncwarp();
    } else if (warp >= kFrontWarp) {
        // ------------------------------------------------------------ MMA issuers
        constexpr uint32_t kIdescS = idesc_bf16_f32(128, NT, 0);  // K-major x K-major
        constexpr uint32_t kIdescG = idesc_bf16_f32(128, D, 1);   // TMEM x MN-major, D wide
        const uint32_t on = elect_one() ? 1u : 0u;
        // MN-major operands step by a chunk from 64 columns to the next 64 (leading dimension).
        const uint64_t desc_base = smem_desc_sw128(smem_addr(smem), 16, 1024);
        const uint32_t desc_hi = (uint32_t)(desc_base >> 32);
        const uint32_t lo0 = (uint32_t)desc_base;
        const uint32_t lo0_mn = (uint32_t)smem_desc_sw128(smem_addr(smem), C::kYChunk, 1024);
        // The rows of -lse and -D terms: K-major without swizzle, 8-row groups 128 bytes apart. The
        // ones have their zeros (K 8..15) a leading-dimension step away; the streamed rows have
        // none, their step is 0: against those zeros any finite value will do.
        const uint32_t aug_hi = (uint32_t)((128 >> 4) | (1u << 14));
        const uint32_t ones_d = (smem_addr(smem + C::kOffOnes) >> 4) | ((4096u >> 4) << 16);
        const uint32_t ones_s = ((smem_addr(smem + C::kOffOnes) + 2048) >> 4) | ((2048u >> 4) << 16);
        const uint32_t vec_lo = smem_addr(smem + C::kOffVec) >> 4;
        const int role = warp - kFrontWarp;  // 0 S, 1 dP, 2 accumulations
        uint32_t n = 0, st = 0, par = 0;     // step, its stage and the stage's parity
        int n_it = 0;
        bool ok = true;
        for (int place = blockIdx.x; place < p.places && ok; place += gridDim.x) {
            const int item = item_at<kDQ>(p, place);
            if (item >= p.items) continue;
            Item it;
            decode<D, kDQ>(p, item, it);
            if (it.steps == 0) continue;
            const int lead = it.lead, last = lead + it.steps - 1;
            if (role < 2) {
                if (!(ok = warp_wait(smem_addr(&bars->x_full), (uint32_t)n_it & 1u, ctl, kSiteFrontX))) break;
                tc_fence_after();
            }
            for (int s = 0; s <= last; ++s, ++n) {
                const uint32_t buf = n & (kBufs - 1), use = n / kBufs;
                const uint32_t y = lo0 + (C::kOffY >> 4) + st * (2 * C::kYTile >> 4);
                if (role == 0) {
                    // S of the step, once the accumulations of four steps before have read the buffer.
                    if (!(ok = warp_wait(smem_addr(&bars->y_full[st]), par, ctl, kSiteFrontY))) break;
                    if (use > 0 && !(ok = warp_wait(smem_addr(&bars->buf_free[buf]), (use - 1) & 1u, ctl, kSiteFrontS))) break;
                    tc_fence_after();
#pragma unroll
                    for (int kk = 0; kk < D / 16; ++kk)
                        umma_ss_on(on, tmem + buf * NT, lo0 + (C::kOffX >> 4) + (kk >> 2) * (C::kXChunk >> 4) + (kk & 3) * 2,
                                   y + (kk >> 2) * (C::kYChunk >> 4) + (kk & 3) * 2, desc_hi, kIdescS, kk > 0);
                    if constexpr (!kDQ) umma_ss_on(on, tmem + buf * NT, ones_s, vec_lo + st * (C::kVec >> 4), aug_hi, kIdescS, 1);
                    umma_commit_on(on, smem_addr(&bars->s_full[buf]));
                    if (s == last) umma_commit_on(on, smem_addr(&bars->x_empty));
                } else if (role == 1) {
                    // dP over S, once the group has loaded S.
                    if (!(ok = warp_wait(smem_addr(&bars->y_full[st]), par, ctl, kSiteFrontY))) break;
                    if (!(ok = warp_wait(smem_addr(&bars->s_read[buf]), use & 1u, ctl, kSiteFrontDP))) break;
                    tc_fence_after();
#pragma unroll
                    for (int kk = 0; kk < D / 16; ++kk)
                        umma_ss_on(on, tmem + buf * NT,
                                   lo0 + ((C::kOffX + C::kXTile) >> 4) + (kk >> 2) * (C::kXChunk >> 4) + (kk & 3) * 2,
                                   y + (C::kYTile >> 4) + (kk >> 2) * (C::kYChunk >> 4) + (kk & 3) * 2, desc_hi, kIdescS,
                                   kk > 0);
                    if constexpr (!kDQ) umma_ss_on(on, tmem + buf * NT, ones_d, vec_lo + st * (C::kVec >> 4), aug_hi, kIdescS, 1);
                    umma_commit_on(on, smem_addr(&bars->dp_full[buf]));
                    if (s == last) umma_commit_on(on, smem_addr(&bars->x_empty));
                } else {
                    if (!(ok = warp_wait(smem_addr(&bars->p_ready[buf]), use & 1u, ctl, kSiteAccP))) break;
                    if (s == 0 && n_it > 0 &&
                        !(ok = warp_wait(smem_addr(&bars->acc_free), (uint32_t)(n_it - 1) & 1u, ctl, kSiteAccFree)))
                        break;
                    tc_fence_after();
                    const uint32_t a_col = tmem + buf * NT, acc = tmem + kColAcc;
                    const uint32_t ymn = lo0_mn + (C::kOffY >> 4) + st * (2 * C::kYTile >> 4);
                    const uint32_t act = s >= lead ? on : 0u;
#pragma unroll
                    for (int kk = 0; kk < NT / 16; ++kk) {  // 16 rows of 128 bytes, 8 TMEM columns
                        const uint32_t add = (s > lead || kk > 0) ? 1u : 0u;
                        if constexpr (kDQ) {
                            umma_ts_on(act, acc, a_col + kk * 8, ymn + kk * 128, desc_hi, kIdescG, add);
                        } else {
                            umma_ts_on(act, acc, a_col + kk * 8, ymn + (C::kYTile >> 4) + kk * 128, desc_hi, kIdescG, add);
                            umma_ts_on(act, acc + D, a_col + NT / 2 + kk * 8, ymn + kk * 128, desc_hi, kIdescG, add);
                        }
                    }
                    umma_commit_on(on, smem_addr(&bars->buf_free[buf]));
                    umma_commit_on(on, smem_addr(&bars->y_empty[st]));
                    if (s == last) umma_commit_on(on, smem_addr(&bars->acc_full));
                }
                __syncwarp();
                if (++st == C::kStages) {
                    st = 0;
                    par ^= 1u;
                }
            }
            ++n_it;
        }
        // Drain: every MMA this warp issued has finished before TMEM is released.
        const uint32_t drain_bar = smem_addr(&bars->drain[role]);
        umma_commit_on(on, drain_bar);
        __syncwarp();
        int never = 0;
        const WaitCtl drain{&never, nullptr, ctl.limit_ns};
        mbar_wait(drain_bar, 0u, drain, 0);
        __syncwarp();
    }

    tc_fence_before();
    __syncthreads();
    if (warp == kFrontWarp) {
        tc_fence_after();
        tmem_dealloc(tmem, kTmemCols);
    }
}

// -lse log2(e), -D, D_r = sum_c dO_rc O_rc, and both as terms (Params::aug), over [B Hq, n_pad].
// Padded rows and rows that saw nothing (lse = -inf) get -inf, and as a term -10^37 (times 0
// it stays 0), so that their weights are 0. D / 8 lanes a row, 16 bytes each.
constexpr int kPrepRows = 4;  // rows of a thread
template <int D>
__global__ void __launch_bounds__(256) prep_kernel(const __nv_bfloat16* __restrict__ o, const char* __restrict__ dout,
                                                   long long sb, long long sh, long long sn, const float* __restrict__ lse,
                                                   float* __restrict__ nlse2, float* __restrict__ nd, uint4* __restrict__ aug,
                                                   float inv_scale, int hq, int n, int n_pad, int with_d) {
    griddep_launch_dependents();
    griddep_wait();
    constexpr int L = D / 8;
    constexpr int R = 256 / L;  // rows of a block's pass
    const int lane = threadIdx.x % L;
    const int bh = blockIdx.x, b = bh / hq, h = bh - b * hq;
    const __nv_bfloat16* o_bh = o + (size_t)bh * n * D + lane * 8;
    const char* d_bh = dout + b * sb + h * sh + lane * 16;
    for (int i0 = (int)(blockIdx.y * R * kPrepRows + threadIdx.x / L); i0 < n_pad; i0 += (int)gridDim.y * R * kPrepRows) {
        // All of a thread's loads before the first sum.
        uint4 x[kPrepRows], y[kPrepRows];
#pragma unroll
        for (int k = 0; k < kPrepRows; ++k) {
            const int i = i0 + k * R;
            x[k] = y[k] = make_uint4(0, 0, 0, 0);
            if (i < n && with_d) {
                x[k] = *reinterpret_cast<const uint4*>(o_bh + (size_t)i * D);
                y[k] = *reinterpret_cast<const uint4*>(d_bh + (long long)i * sn);
            }
        }
        float mine = 0.f;  // lane k's: the sum of row k
#pragma unroll
        for (int k = 0; k < kPrepRows; ++k) {
            float acc = 0.f;
            const uint32_t xs[4] = {x[k].x, x[k].y, x[k].z, x[k].w}, ys[4] = {y[k].x, y[k].y, y[k].z, y[k].w};
#pragma unroll
            for (int c = 0; c < 4; ++c)
                acc += __uint_as_float(xs[c] << 16) * __uint_as_float(ys[c] << 16) +
                       __uint_as_float(xs[c] & 0xffff0000u) * __uint_as_float(ys[c] & 0xffff0000u);
#pragma unroll
            for (int m = L / 2; m > 0; m >>= 1) acc += __shfl_xor_sync(0xffffffffu, acc, m);
            if (lane == k) mine = acc;
        }
        if (lane < kPrepRows) {
            const int i = i0 + lane * R;  // n_pad is a multiple of 128, and so of a pass: all rows or none
            const float l = i < n ? lse[(size_t)bh * n + i] : -INFINITY;
            const bool seen = l != -INFINITY;
            const size_t r = (size_t)bh * n_pad + i;
            nlse2[r] = seen ? -l * 1.4426950408889634f : -INFINITY;
            nd[r] = -mine;
            uint32_t l0, l1, l2, d0, d1, d2;
            split3(seen ? -l * inv_scale : -1e37f, l0, l1, l2);
            split3(-mine, d0, d1, d2);
            aug[r] = make_uint4(l0 | (l1 << 16), l2 | (d0 << 16), d1 | (d2 << 16), 0u);
        }
    }
}

// Sums the parts of dV and dK of the tiles [j0, j0 + tiles) in their order.
template <int D>
__global__ void __launch_bounds__(256) join_kernel(const float* __restrict__ part, __nv_bfloat16* __restrict__ dk,
                                                   __nv_bfloat16* __restrict__ dv, int j0, int tiles, int splits, int n_kv,
                                                   long long units) {
    griddep_launch_dependents();
    griddep_wait();
    const long long total = units * tiles * 2 * 128 * (D / 4);
    const long long k = (long long)blockIdx.x * 256 + threadIdx.x;
    if (k >= total) return;
    const int c = (int)(k % (D / 4)) * 4;
    long long rest = k / (D / 4);
    const int row = (int)(rest % 128);
    rest /= 128;
    const int which = (int)(rest % 2);
    rest /= 2;
    const int t = (int)(rest % tiles);
    const long long unit = rest / tiles;
    const int key = (j0 + t) * 128 + row;
    if (key >= n_kv) return;
    float4 s = make_float4(0.f, 0.f, 0.f, 0.f);
    for (int x = 0; x < splits; ++x) {
        const long long slot = (unit * tiles + t) * splits + x;
        const float4 a = *reinterpret_cast<const float4*>(part + ((slot * 2 + which) * 128 + row) * D + c);
        s.x += a.x;
        s.y += a.y;
        s.z += a.z;
        s.w += a.w;
    }
    *reinterpret_cast<uint2*>((which ? dk : dv) + (unit * n_kv + key) * D + c) =
        make_uint2(pack_bf16x2(s.x, s.y), pack_bf16x2(s.z, s.w));
}

}  // namespace winb
