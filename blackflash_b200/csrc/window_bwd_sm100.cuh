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
// streams pairs of NT-row tiles Y0, Y1 past them:
//                    X0  X1   Y0  Y1    S = X0 Y0^T   dP = X1 Y1^T   accumulators
//   dK/dV (kDQ=0)    K   V    Q   dO    (S^T)         (dP^T)         dV += P^T Y1, dK += dS^T Y0
//   dQ    (kDQ=1)    Q   dO   K   V                                  dQ += dS Y0
// D. Both passes read it from an array that the prep kernel fills from O. O is rounded to
// bf16, and for a row that sees few keys that error is not small against dP - D, of which D
// is then a large part (one key: dP - D is 0). So with few keys (two_sweeps) the dQ pass
// walks its KV tiles twice: first it sums P dP and P in fp32, D = sum P dP / sum P, which it
// also leaves in the array for the dK/dV pass; then it accumulates.
// Roles: eight elementwise warps (two threads per row), a TMA producer, an issuer of S and
// dP, an issuer of the accumulations; persistent blocks, so an item's tail overlaps the next
// one's first products. S has two buffers: S of step n + 1 is computed while the elementwise
// warps are at step n. P and dS go back to TMEM as bf16, over the S buffer they came from,
// and are the A operands of the accumulations; neither leaves the SM.
// TMEM (512 columns):  dK/dV d=64: S 2x128, dP 128, dV 64, dK 64
//                      dK/dV d=128: NT = 64 queries: S 2x64, dP 2x64, dV 128, dK 128
//                      dQ: S 2x128, dP 128, dQ 64 / 128
namespace winb {

using win::kTmemCols;

constexpr int kThreads = 12 * 32;
constexpr int kEwWarps = 8;
constexpr int kProdWarp = 8;
constexpr int kFrontWarp = 9;  // issues S and dP; owns the TMEM allocation
constexpr int kAccWarp = 10;   // issues the accumulations; warp 11 completes the warpgroup
constexpr int kEwRegs = 216, kOtherRegs = 64;  // launch budget 384 x 168
static_assert(kEwWarps * 32 * kEwRegs + 128 * kOtherRegs <= kThreads * 168, "register split exceeds the launch budget");

template <int D, bool kDQ>
struct Cfg {
    static constexpr int NT = !kDQ && D == 128 ? 64 : 128;  // rows of a streamed tile
    static constexpr int kChunks = D / 64;
    static constexpr int kXChunk = 128 * 128, kXTile = kChunks * kXChunk;
    static constexpr int kYChunk = NT * 128, kYTile = kChunks * kYChunk;
    static constexpr int kStages = kDQ && D == 128 ? 2 : 4;
    static constexpr int kVec = kDQ ? 0 : 2 * NT * 4;  // -lse2 and -D of the streamed queries
    static constexpr int kOffX = 0;
    static constexpr int kOffY = kOffX + 2 * kXTile;              // [kStages][Y0, Y1]
    static constexpr int kOffVec = kOffY + kStages * 2 * kYTile;  // [kStages]
    static constexpr int kOffBar = kOffVec + kStages * kVec;
    static constexpr int kDpBufs = NT == 64 ? 2 : 1;
    static constexpr int kColDP = 2 * NT;
    static constexpr int kColAcc = kColDP + kDpBufs * NT;
    static constexpr int kAccs = kDQ ? 1 : 2;
    static_assert(kColAcc + kAccs * D <= kTmemCols, "TMEM columns");
};

template <int D, bool kDQ>
struct Bars {
    uint64_t x_full, x_empty;
    uint64_t y_full[Cfg<D, kDQ>::kStages], y_empty[Cfg<D, kDQ>::kStages];
    uint64_t s_full[2], s_free[2], p_ready[2];
    uint64_t dp_full[2], dp_free[2];
    uint64_t acc_full, acc_free;
    uint64_t drain[2];
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
};

struct Params {
    int items;
    int batch, hq, hkv, group;
    int n_q, n_kv, n_pad;    // n_pad: n_q rounded up to 128, row stride of nlse2 / nd
    int nk, ns;              // KV tiles; of them tiles that hold sinks
    int window, sinks;       // clamped to n_kv
    int q_tiles;             // 128-row query tiles (dQ)
    int splits_s, splits_n;  // dK/dV: parts of a sink tile's and of another tile's queries
    float scale, scale_log2;
    const float* nlse2;      // [B Hq, n_pad] -lse log2(e); -inf past n_q and for rows that see nothing
    float* nd;               // [B Hq, n_pad] -D
    int two_sweeps;          // dQ: find D in a first sweep over the KV tiles, and store it
    __nv_bfloat16 *dq, *dk, *dv;
    float* part;             // [slot][dV, dK][128][D] of the tiles with more than one part
    unsigned long long timeout_ns;
};

struct Item {
    int b, kvh, head;   // head: the query head (dQ)
    int tile;           // stationary 128-row tile
    int steps;          // dQ: of one sweep
    int i0, ni, s0;     // dK/dV: step s is query tile i0 + (s0 + s) % ni of head (s0 + s) / ni
    int n_sink, skip;   // dQ: step s is KV tile s, or s + skip past the sink tiles
    long long slot;     // dK/dV: part to write, -1: the gradient itself
};

// First query tile and number of query tiles (NT rows) that see KV tile j.
template <int NT>
__device__ __forceinline__ void queries_of(const Params& p, int j, int& i0, int& ni) {
    const int off = p.n_kv - p.n_q;
    const int last_key = min(j * 128 + 127, p.n_kv - 1);
    const int lo = max(0, j * 128 - off);
    const int hi = j < p.ns ? p.n_q : min(p.n_q, last_key + p.window - off);
    i0 = lo / NT;
    ni = hi > lo ? (hi + NT - 1) / NT - i0 : 0;
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
        const int lo = max(0, p_first - p.window + 1) >> 7;
        const int hi = p_last >= 0 ? (p_last >> 7) + 1 : 0;
        it.n_sink = min(p.ns, lo);
        it.skip = lo - it.n_sink;
        it.steps = hi > 0 ? hi - it.skip : 0;
        it.slot = -1;
    } else {
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
        queries_of<Cfg<D, kDQ>::NT>(p, it.tile, it.i0, it.ni);
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
    constexpr int NT = C::NT;
    constexpr int NC = NT / 2;  // streamed rows (S columns) of a thread
    extern __shared__ uint8_t smem_raw[];
    uint8_t* smem = align1024(smem_raw);
    Bars<D, kDQ>* bars = reinterpret_cast<Bars<D, kDQ>*>(smem + C::kOffBar);
    const int warp = threadIdx.x >> 5;
    const int lane = threadIdx.x & 31;

    if (threadIdx.x == 0) {
        mbar_init(smem_addr(&bars->x_full), 1);
        mbar_init(smem_addr(&bars->x_empty), 1);
        for (int s = 0; s < C::kStages; ++s) {
            mbar_init(smem_addr(&bars->y_full[s]), 1);
            mbar_init(smem_addr(&bars->y_empty[s]), 1);
        }
        for (int b = 0; b < 2; ++b) {
            mbar_init(smem_addr(&bars->s_full[b]), 1);
            mbar_init(smem_addr(&bars->s_free[b]), 1);
            mbar_init(smem_addr(&bars->p_ready[b]), kEwWarps);  // one arrival per elementwise warp
            mbar_init(smem_addr(&bars->dp_full[b]), 1);
            mbar_init(smem_addr(&bars->dp_free[b]), kEwWarps);
            mbar_init(smem_addr(&bars->drain[b]), 1);
        }
        mbar_init(smem_addr(&bars->acc_full), 1);
        mbar_init(smem_addr(&bars->acc_free), kEwWarps);
        bars->abort_flag = 0;
        fence_barrier_init();
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
        const int quarter = warp & 3;
        const int sub = warp >> 2;
        const int h = lane >> 4;                                // S columns NC h .. NC h + NC - 1
        const int row = quarter * 32 + sub * 16 + (lane & 15);  // row of the tile == TMEM lane
        const uint32_t tl = tmem + ((uint32_t)(quarter * 32 + sub * 16) << 16);
        const int off = p.n_kv - p.n_q;
        const uint64_t sl2_2 = f2_pack(p.scale_log2, p.scale_log2);
        uint32_t n = 0;  // steps so far
        int n_it = 0;    // items with steps so far
        bool ok = true;
        for (int item = blockIdx.x; item < p.items && ok; item += gridDim.x) {
            Item it;
            decode<D, kDQ>(p, item, it);
            const int xrow = it.tile * 128 + row;
            // dQ: the row's -lse2 and -D (padded rows have entries).
            const int lead = kDQ && p.two_sweeps ? it.steps : 0;  // steps of the first sweep
            const size_t at = kDQ ? ((size_t)it.b * p.hq + it.head) * p.n_pad + xrow : 0;
            uint64_t nl2 = 0, nd2 = 0;
            float sum_p = 0.f, sum_pdp = 0.f;
            if constexpr (kDQ) {
                const float a = p.nlse2[at], b = lead ? 0.f : p.nd[at];
                nl2 = f2_pack(a, a);
                nd2 = f2_pack(b, b);
            }
            for (int s_all = 0; s_all < lead + it.steps; ++s_all, ++n) {
                const bool measure = kDQ && s_all < lead;
                const int s_i = measure || !kDQ ? s_all : s_all - lead;
                if (kDQ && lead && s_all == lead) {
                    // The two halves of the row; a row that sees nothing has D = 0.
                    sum_p += __shfl_xor_sync(0xffffffffu, sum_p, 16);
                    sum_pdp += __shfl_xor_sync(0xffffffffu, sum_pdp, 16);
                    const float b = sum_p != 0.f ? -sum_pdp / sum_p : 0.f;
                    nd2 = f2_pack(b, b);
                    if (h == 0) p.nd[at] = b;
                }
                const int buf = n & 1;
                const uint32_t tS = tl + (uint32_t)(buf * NT);
                // Visible: column c with c < last and (c >= first or c < snk).
                int first, last, snk;
                if constexpr (kDQ) {
                    const int c0 = (s_i < it.n_sink ? s_i : s_i + it.skip) * 128 + h * NC;
                    last = xrow + off + 1 - c0;
                    first = xrow + off + 1 - p.window - c0;
                    snk = p.sinks - c0;
                } else {
                    const int q0 = (it.i0 + (it.s0 + s_i) % it.ni) * NT + h * NC;
                    first = xrow - off - q0;
                    last = xrow < p.sinks ? NC : first + p.window;
                    snk = 0;
                }
                if (!(ok = warp_wait(smem_addr(&bars->s_full[buf]), (n >> 1) & 1u, ctl, kSiteEwS))) break;
                tc_fence_after();
                float pr[NC];
                {
                    uint32_t s[NC / 32][32];
#pragma unroll
                    for (int i = 0; i < NC / 32; ++i) tmem_ld16x32bx2_x32<NC>(tS + 32 * i, s[i]);
                    tmem_wait_ld();
#pragma unroll
                    for (int c = 0; c < NC; ++c) pr[c] = __uint_as_float(s[c >> 5][c & 31]);
                }
                if constexpr (!kDQ) {
                    // The vectors came with Y; seen here too, their copy is visible to this warp.
                    if (!(ok = warp_wait(smem_addr(&bars->y_full[n % C::kStages]), (n / C::kStages) & 1u, ctl, kSiteEwS))) break;
                }
                if (last < NC || (first > 0 && snk < NC)) {
#pragma unroll
                    for (int c = 0; c < NC; ++c)
                        if (c >= last || (c < first && c >= snk)) pr[c] = -INFINITY;
                }
                const float* vec = reinterpret_cast<const float*>(smem + C::kOffVec + (n % C::kStages) * C::kVec) + h * NC;
#pragma unroll
                for (int c = 0; c < NC; c += 4) {
                    uint64_t a = nl2, b = nl2;
                    if constexpr (!kDQ) {
                        const float4 v = *reinterpret_cast<const float4*>(vec + c);
                        a = f2_pack(v.x, v.y);
                        b = f2_pack(v.z, v.w);
                    }
                    float x0, x1, x2, x3;
                    f2_unpack(f2_fma(f2_pack(pr[c], pr[c + 1]), sl2_2, a), x0, x1);
                    f2_unpack(f2_fma(f2_pack(pr[c + 2], pr[c + 3]), sl2_2, b), x2, x3);
                    pr[c] = fast_exp2(x0);
                    pr[c + 1] = fast_exp2(x1);
                    pr[c + 2] = fast_exp2(x2);
                    pr[c + 3] = fast_exp2(x3);
                }
                if constexpr (!kDQ) {
                    // P^T as bf16 over S's first half (this thread: words NC h / 2 ..).
#pragma unroll
                    for (int i = 0; i < NC / 32; ++i) {
                        uint32_t pk[16];
#pragma unroll
                        for (int c = 0; c < 16; ++c) pk[c] = pack_bf16x2(pr[32 * i + 2 * c], pr[32 * i + 2 * c + 1]);
                        tmem_st16x32bx2_x16<NC / 2>(tS + 16 * i, pk);
                    }
                }
                // dS = P (dP - D)
                const int db = C::kDpBufs == 2 ? buf : 0;
                const uint32_t dpar = (C::kDpBufs == 2 ? n >> 1 : n) & 1u;
                if (!(ok = warp_wait(smem_addr(&bars->dp_full[db]), dpar, ctl, kSiteEwDP))) break;
                tc_fence_after();
                uint32_t dsk[NC / 2];
#pragma unroll
                for (int i = 0; i < NC / 32; ++i) {
                    uint32_t dp[32];
                    tmem_ld16x32bx2_x32<NC>(tl + C::kColDP + db * NT + 32 * i, dp);
                    tmem_wait_ld();
                    if (i == NC / 32 - 1) {  // dP is in registers: the next one may be computed
                        tc_fence_before();
                        __syncwarp();
                        if (lane == 0) mbar_arrive(smem_addr(&bars->dp_free[db]));
                    }
#pragma unroll
                    for (int c = 0; c < 32; c += 4) {
                        uint64_t a = nd2, b = nd2;
                        if constexpr (!kDQ) {
                            const float4 v = *reinterpret_cast<const float4*>(vec + NT + 32 * i + c);
                            a = f2_pack(v.x, v.y);
                            b = f2_pack(v.z, v.w);
                        }
                        float x0, x1, x2, x3;
                        f2_unpack(f2_add(f2_pack(__uint_as_float(dp[c]), __uint_as_float(dp[c + 1])), a), x0, x1);
                        f2_unpack(f2_add(f2_pack(__uint_as_float(dp[c + 2]), __uint_as_float(dp[c + 3])), b), x2, x3);
                        if (kDQ && measure) {  // D is 0 so far: x is dP
                            const float* q = pr + 32 * i + c;
                            sum_p += (q[0] + q[1]) + (q[2] + q[3]);
                            sum_pdp += (q[0] * x0 + q[1] * x1) + (q[2] * x2 + q[3] * x3);
                        }
                        dsk[16 * i + c / 2] = pack_bf16x2(pr[32 * i + c] * x0, pr[32 * i + c + 1] * x1);
                        dsk[16 * i + c / 2 + 1] = pack_bf16x2(pr[32 * i + c + 2] * x2, pr[32 * i + c + 3] * x3);
                    }
                }
                if (!measure) {
#pragma unroll
                    for (int i = 0; i < NC / 32; ++i)
                        tmem_st16x32bx2_x16<NC / 2>(tS + (kDQ ? 0 : NT / 2) + 16 * i, dsk + 16 * i);
                    tmem_wait_st();
                }
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(smem_addr(&bars->p_ready[buf]));
            }
            if (!ok) break;

            // ---------------------------------------------------- the item's gradients
            const bool any = it.steps > 0;
            if (any) {
                if (!(ok = warp_wait(smem_addr(&bars->acc_full), (uint32_t)n_it & 1u, ctl, kSiteEwAcc))) break;
                ++n_it;
                tc_fence_after();
            }
#pragma unroll 1
            for (int i = 0; i < C::kAccs * (D / 64); ++i) {
                const int which = i / (D / 64), part = i % (D / 64);  // dK/dV: 0 dV, 1 dK
                uint32_t o[32];
                if (any) {
                    tmem_ld16x32bx2_x32<D / 2>(tl + C::kColAcc + which * D + 32 * part, o);
                    tmem_wait_ld();
                } else {
#pragma unroll
                    for (int c = 0; c < 32; ++c) o[c] = 0u;
                }
                const int col = h * (D / 2) + 32 * part;
                const float f = kDQ || which ? p.scale : 1.f;
                if (it.slot >= 0) {
                    float4* dst = reinterpret_cast<float4*>(p.part + ((it.slot * 2 + which) * 128 + row) * D + col);
#pragma unroll
                    for (int c = 0; c < 8; ++c)
                        dst[c] = make_float4(__uint_as_float(o[4 * c]) * f, __uint_as_float(o[4 * c + 1]) * f,
                                             __uint_as_float(o[4 * c + 2]) * f, __uint_as_float(o[4 * c + 3]) * f);
                } else if (xrow < (kDQ ? p.n_q : p.n_kv)) {
                    __nv_bfloat16* base = kDQ ? p.dq + (((size_t)it.b * p.hq + it.head) * p.n_q + xrow) * D
                                              : (which ? p.dk : p.dv) + (((size_t)it.b * p.hkv + it.kvh) * p.n_kv + xrow) * D;
                    uint4* dst = reinterpret_cast<uint4*>(base + col);
#pragma unroll
                    for (int c = 0; c < 4; ++c) {
                        uint32_t w[4];
#pragma unroll
                        for (int e = 0; e < 4; ++e)
                            w[e] = pack_bf16x2(__uint_as_float(o[8 * c + 2 * e]) * f, __uint_as_float(o[8 * c + 2 * e + 1]) * f);
                        dst[c] = make_uint4(w[0], w[1], w[2], w[3]);
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
        for (int item = blockIdx.x; item < p.items && ok; item += gridDim.x) {
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
            const int lead = kDQ && p.two_sweeps ? it.steps : 0;
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
                        const int s = it.s0 + s_i;
                        yrow = (it.i0 + s % it.ni) * NT;
                        head = it.kvh * p.group + s / it.ni;
                    }
                    mbar_arrive_expect_tx(f, 2 * C::kYTile + C::kVec);
                    const uint32_t y = y0 + (uint32_t)(st * 2 * C::kYTile);
                    for (int ch = 0; ch < C::kChunks; ++ch) {
                        tma_load_4d(y + ch * C::kYChunk, &tmY0, f, ch * 64, yrow, head, it.b);
                        tma_load_4d(y + C::kYTile + ch * C::kYChunk, &tmY1, f, ch * 64, yrow, head, it.b);
                    }
                    if constexpr (!kDQ) {
                        const size_t at = ((size_t)it.b * p.hq + head) * p.n_pad + yrow;
                        bulk_load(vec0 + st * C::kVec, p.nlse2 + at, NT * 4, f);
                        bulk_load(vec0 + st * C::kVec + NT * 4, p.nd + at, NT * 4, f);
                    }
                }
                __syncwarp();
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
    } else if (warp == kFrontWarp || warp == kAccWarp) {
        // ------------------------------------------------------------ MMA issuers
        constexpr uint32_t kIdescS = idesc_bf16_f32(128, NT, 0);  // K-major x K-major
        constexpr uint32_t kIdescG = idesc_bf16_f32(128, 64, 1);  // TMEM x MN-major 64-column chunk
        const bool leader = elect_one();
        const uint64_t desc_base = smem_desc_sw128(smem_addr(smem), 16, 1024);
        const uint32_t desc_hi = (uint32_t)(desc_base >> 32);
        const uint32_t lo0 = (uint32_t)desc_base;
        const uint32_t x_lo = lo0 + (C::kOffX >> 4), y_lo0 = lo0 + (C::kOffY >> 4);
        const bool front = warp == kFrontWarp;
        uint32_t n = 0;
        int n_it = 0, st = 0;
        uint32_t par = 0;
        bool ok = true;
        for (int item = blockIdx.x; item < p.items && ok; item += gridDim.x) {
            Item it;
            decode<D, kDQ>(p, item, it);
            if (it.steps == 0) continue;
            if (front) {
                if (!(ok = warp_wait(smem_addr(&bars->x_full), (uint32_t)n_it & 1u, ctl, kSiteFrontX))) break;
                tc_fence_after();
            }
            const int lead = kDQ && p.two_sweeps ? it.steps : 0, last = lead + it.steps - 1;
            for (int s_i = 0; s_i <= last; ++s_i, ++n) {
                const int buf = n & 1;
                const uint32_t y_lo = y_lo0 + (uint32_t)(st * 2 * C::kYTile >> 4);
                const uint32_t tS = tmem + (uint32_t)(buf * NT);
                if (front) {
                    if (!(ok = warp_wait(smem_addr(&bars->y_full[st]), par, ctl, kSiteFrontY))) break;
                    if (n >= 2 && !(ok = warp_wait(smem_addr(&bars->s_free[buf]), ((n >> 1) - 1) & 1u, ctl, kSiteFrontS))) break;
                    tc_fence_after();
                    if (leader) {
#pragma unroll
                        for (int kk = 0; kk < D / 16; ++kk)
                            umma_ss_lo(tS, x_lo + (uint32_t)(kk >> 2) * (C::kXChunk >> 4) + (uint32_t)(kk & 3) * 2,
                                       y_lo + (uint32_t)(kk >> 2) * (C::kYChunk >> 4) + (uint32_t)(kk & 3) * 2, desc_hi,
                                       kIdescS, kk > 0);
                        umma_commit(smem_addr(&bars->s_full[buf]));
                    }
                    __syncwarp();
                    const int db = C::kDpBufs == 2 ? buf : 0;
                    const uint32_t uses = C::kDpBufs == 2 ? n >> 1 : n;  // earlier uses of this dP buffer
                    if (uses > 0 && !(ok = warp_wait(smem_addr(&bars->dp_free[db]), (uses - 1) & 1u, ctl, kSiteFrontDP))) break;
                    tc_fence_after();
                    if (leader) {
#pragma unroll
                        for (int kk = 0; kk < D / 16; ++kk)
                            umma_ss_lo(tmem + C::kColDP + db * NT,
                                       x_lo + (C::kXTile >> 4) + (uint32_t)(kk >> 2) * (C::kXChunk >> 4) + (uint32_t)(kk & 3) * 2,
                                       y_lo + (C::kYTile >> 4) + (uint32_t)(kk >> 2) * (C::kYChunk >> 4) + (uint32_t)(kk & 3) * 2,
                                       desc_hi, kIdescS, kk > 0);
                        umma_commit(smem_addr(&bars->dp_full[db]));
                        if (s_i == last) umma_commit(smem_addr(&bars->x_empty));
                    }
                    __syncwarp();
                } else {
                    if (!(ok = warp_wait(smem_addr(&bars->p_ready[buf]), (n >> 1) & 1u, ctl, kSiteAccP))) break;
                    if (s_i == 0 && n_it > 0 &&
                        !(ok = warp_wait(smem_addr(&bars->acc_free), (uint32_t)(n_it - 1) & 1u, ctl, kSiteAccFree)))
                        break;
                    tc_fence_after();
                    if (leader && s_i >= lead) {
                        const uint32_t acc = tmem + C::kColAcc;
#pragma unroll
                        for (int kk = 0; kk < NT / 16; ++kk)
#pragma unroll
                            for (int ch = 0; ch < C::kChunks; ++ch) {
                                const uint32_t off = ch * (C::kYChunk >> 4) + kk * 128;  // 16 rows of 128 bytes
                                const uint32_t add = (s_i > lead || kk > 0) ? 1u : 0u;
                                if constexpr (kDQ) {
                                    umma_ts_lo(acc + ch * 64, tS + kk * 8, y_lo + off, desc_hi, kIdescG, add);
                                } else {
                                    umma_ts_lo(acc + ch * 64, tS + kk * 8, y_lo + (C::kYTile >> 4) + off, desc_hi, kIdescG, add);
                                    umma_ts_lo(acc + D + ch * 64, tS + NT / 2 + kk * 8, y_lo + off, desc_hi, kIdescG, add);
                                }
                            }
                    }
                    if (leader) {
                        umma_commit(smem_addr(&bars->s_free[buf]));
                        umma_commit(smem_addr(&bars->y_empty[st]));
                        if (s_i == last) umma_commit(smem_addr(&bars->acc_full));
                    }
                    __syncwarp();
                }
                if (++st == C::kStages) {
                    st = 0;
                    par ^= 1u;
                }
            }
            ++n_it;
        }
        // Drain: every MMA this warp issued has finished before TMEM is released.
        const uint32_t drain_bar = smem_addr(&bars->drain[front ? 0 : 1]);
        if (leader) umma_commit(drain_bar);
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

// -lse log2(e) and -D, D_r = sum_c dO_rc O_rc, over [B Hq, n_pad]. Padded rows and rows that
// saw nothing (lse = -inf) get -inf, so that exp2(s + that) = 0. Eight lanes a row of 64.
template <int D>
__global__ void __launch_bounds__(256) prep_kernel(const __nv_bfloat16* __restrict__ o, const char* __restrict__ dout,
                                                   long long sb, long long sh, long long sn, const float* __restrict__ lse,
                                                   float* __restrict__ nlse2, float* __restrict__ nd, int hq, int n,
                                                   int n_pad, long long rows, int with_d) {
    griddep_launch_dependents();
    griddep_wait();
    constexpr int L = D / 8;  // lanes of a row, 16 bytes each
    const int lane = threadIdx.x % L;
    const long long r = ((long long)blockIdx.x * 256 + threadIdx.x) / L;
    const bool live = r < rows;
    const long long bh = live ? r / n_pad : 0;
    const int i = (int)(r - bh * n_pad);
    const bool in = live && i < n;
    float acc = 0.f;
    if (in && with_d) {
        const long long b = bh / hq, h = bh - b * hq;
        const uint4 x = *reinterpret_cast<const uint4*>(o + (bh * n + i) * D + lane * 8);
        const uint4 y = *reinterpret_cast<const uint4*>(dout + b * sb + h * sh + i * sn + lane * 16);
        const uint32_t xs[4] = {x.x, x.y, x.z, x.w}, ys[4] = {y.x, y.y, y.z, y.w};
#pragma unroll
        for (int c = 0; c < 4; ++c)
            acc += __uint_as_float(xs[c] << 16) * __uint_as_float(ys[c] << 16) +
                   __uint_as_float(xs[c] & 0xffff0000u) * __uint_as_float(ys[c] & 0xffff0000u);
    }
#pragma unroll
    for (int m = L / 2; m > 0; m >>= 1) acc += __shfl_xor_sync(0xffffffffu, acc, m);
    if (live && lane == 0) {
        const float l = in ? lse[bh * n + i] : -INFINITY;
        nlse2[r] = l == -INFINITY ? -INFINITY : -l * 1.4426950408889634f;
        nd[r] = -acc;
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
