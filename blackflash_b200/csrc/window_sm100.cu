// Sliding-window attention with sinks: forward, backward, and the prefix part of a decoding
// step, which is the same kernel with nothing masked. Host side; the kernels are in
// window_fwd_sm100.cuh and window_bwd_sm100.cuh.
#include <cuda_bf16.h>
#include <math.h>
#include <string.h>

#include "sm100_ptx.cuh"
#include "views.h"

namespace bfk {

// Set by a bounded wait that gave up; read by blackflash_status().
__device__ unsigned int g_wait_status = 0;

__device__ __forceinline__ uint8_t* align1024(uint8_t* p) {
    return reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(p) + 1023) & ~uintptr_t(1023));
}

#include "window_fwd_sm100.cuh"
#include "window_bwd_sm100.cuh"

}  // namespace bfk

namespace {

constexpr unsigned long long kTimeoutNs = 4000000000ull;
constexpr float kLog2e = 1.4426950408889634f;

template <int D, bool kF16, bool kPartial, bool kNarrow>
int launch_fwd(const CUtensorMap& mq, const CUtensorMap& mk, const CUtensorMap& mv, const bfk::win::Params& p,
               cudaStream_t stream) {
    static std::atomic<bool> done[64];  // per device; zero-initialised (static storage)
    auto kernel = bfk::win::window_fwd_kernel<D, kF16, kPartial, kNarrow>;
    int rc, sms = 0;
    if ((rc = allow_smem(kernel, bfk::win::smem_bytes<D>(), done)) != BF_OK) return rc;
    if ((rc = sm_count(&sms)) != BF_OK) return rc;
    const int grid = p.items < sms ? p.items : sms;  // persistent: at most one CTA per SM
    return launch_error(launch_pdl(kernel, dim3((unsigned)grid), bfk::win::kThreads, bfk::win::smem_bytes<D>(), stream, mq,
                                   mk, mv, p));
}

template <bool kPartial, bool kNarrow>
int launch_fwd(int d, bool f16, const CUtensorMap& mq, const CUtensorMap& mk, const CUtensorMap& mv,
               const bfk::win::Params& p, cudaStream_t stream) {
    if (d == 64)
        return f16 ? launch_fwd<64, true, kPartial, kNarrow>(mq, mk, mv, p, stream)
                   : launch_fwd<64, false, kPartial, kNarrow>(mq, mk, mv, p, stream);
    return f16 ? launch_fwd<128, true, kPartial, kNarrow>(mq, mk, mv, p, stream)
               : launch_fwd<128, false, kPartial, kNarrow>(mq, mk, mv, p, stream);
}

int check_window(int B, int Hq, int Hkv, int Nq, int Nkv, int d, int window, int sinks, float scale) {
    if (B <= 0 || Hq <= 0 || Hkv <= 0 || Nq <= 0 || Nkv <= 0)
        return bf_set_error(BF_ERR_ARG, "empty problem: B, H and N must be >= 1");
    if (Hq % Hkv) return bf_set_error(BF_ERR_ARG, "query heads must be a multiple of KV heads");
    if (d != 64 && d != 128) return bf_set_error(BF_ERR_ARG, "BlackFlash supports d=64 and d=128");
    if (Nq > (1 << 30) || Nkv > (1 << 30)) return bf_set_error(BF_ERR_ARG, "more than 2^30 rows");
    if (window < 1 || sinks < 0) return bf_set_error(BF_ERR_ARG, "need window >= 1 and sinks >= 0");
    if (!(scale >= 1e-30f) || !isfinite(scale)) return bf_set_error(BF_ERR_ARG, "scale must be positive (at least 1e-30) and finite");
    return BF_OK;
}

}  // namespace

extern "C" int blackflash_window_fwd(const bf_view* Q, const bf_view* K, const bf_view* V, void* O, float* lse, int B,
                                     int Hq, int Hkv, int Nq, int Nkv, int d, int window, int sinks, float scale, int dtype,
                                     void* stream) {
    bf_set_error(BF_OK, "");
    int rc;
    if ((rc = check_window(B, Hq, Hkv, Nq, Nkv, d, window, sinks, scale)) != BF_OK) return rc;
    if (dtype != BF_DTYPE_BF16 && dtype != BF_DTYPE_F16) return bf_set_error(BF_ERR_ARG, "dtype must be bf16 or fp16");
    ViewStrides sq, sk, sv;
    if ((rc = check_view(Q, "Q", B, Hq, Nq, d, 2, &sq)) != BF_OK) return rc;
    if ((rc = check_view(K, "K", B, Hkv, Nkv, d, 2, &sk)) != BF_OK) return rc;
    if ((rc = check_view(V, "V", B, Hkv, Nkv, d, 2, &sv)) != BF_OK) return rc;
    if (!O || (reinterpret_cast<uintptr_t>(O) & 31u)) return bf_set_error(BF_ERR_ARG, "O must be 32-byte aligned");

    bfk::win::Params p;
    memset(&p, 0, sizeof(p));
    p.batch = B;
    p.hq = Hq;
    p.hkv = Hkv;
    p.group = Hq / Hkv;
    p.n_q = Nq;
    p.n_kv = Nkv;
    p.nk = (Nkv + 127) / 128;
    p.scale_log2 = scale * kLog2e;
    p.out = O;
    p.lse = lse;
    p.timeout_ns = kTimeoutNs;
    p.window = window < Nkv ? window : Nkv;
    p.sinks = sinks < Nkv ? sinks : Nkv;
    p.ns = (p.sinks + 127) / 128;
    p.pair_heads = p.group % 2 == 0;
    const int rows = p.pair_heads ? 128 : 256;
    p.q_blocks = (Nq + rows - 1) / rows;
    const long long units = (long long)B * Hq / (p.pair_heads ? 2 : 1);
    if ((long long)B * Hq > 0x7fffffffLL || units * p.q_blocks > 0x7fffffffLL)
        return bf_set_error(BF_ERR_ARG, "problem too large for one launch");
    p.items = (int)(units * p.q_blocks);
    p.by_units.set((uint32_t)units);
    p.by_heads.set((uint32_t)(p.pair_heads ? Hq / 2 : Hq));
    p.by_group.set((uint32_t)p.group);

    if ((rc = bind_context()) != BF_OK) return rc;
    const bool f16 = dtype == BF_DTYPE_F16;
    CUtensorMap mq, mk, mv;
    const long long dq[4] = {d, Nq, Hq, B}, dk[4] = {d, Nkv, Hkv, B};
    const long long tq[3] = {sq.s[2], sq.s[1], sq.s[0]}, tk[3] = {sk.s[2], sk.s[1], sk.s[0]},
                    tv[3] = {sv.s[2], sv.s[1], sv.s[0]};
    if ((rc = make_map_4d(&mq, Q->data, f16, dq, tq, 128, 1)) != BF_OK) return rc;
    if ((rc = make_map_4d(&mk, K->data, f16, dk, tk, 128, 1)) != BF_OK) return rc;
    if ((rc = make_map_4d(&mv, V->data, f16, dk, tv, 128, 1)) != BF_OK) return rc;
    // Sinks in a step of 32 columns where they fit one: at N = 8192 with 4 sinks, d = 64, window
    // 1024 it takes 235 -> 209 us. At d = 128 the larger kernel's full steps are scheduled worse, so
    // there only for short windows. us full / narrow at d = 128, 4 sinks (1 and 32 alike), by window:
    //                           256          384          512          640          768
    //   B=4 Hq=16 Hkv=4 N=8192  167 / 161    191 / 188    219 / 218    244 / 246    277 / 282
    //   B=2 H=16 N=4096         58.9 / 55.0  66.6 / 63.8  71.9 / 70.7  77.6 / 77.2  83.2 / 83.5
    //   B=4 Hq=8 Hkv=2 N=2048   27.5 / 25.5  31.3 / 29.9  35.2 / 34.0  38.9 / 38.1  40.7 / 41.1
    const bool narrow = p.sinks > 0 && p.sinks <= 32 && (d == 64 || p.window <= 512);
    cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
    return narrow ? launch_fwd<false, true>(d, f16, mq, mk, mv, p, st) : launch_fwd<false, false>(d, f16, mq, mk, mv, p, st);
}

namespace {

// How the dK/dV pass is split, and its workspace: -lse2 and -D, both as terms, then the parts.
struct BwdPlan {
    int nk, ns, window, sinks, n_pad, splits_s, splits_n;
    int times;  // a sink tile's part has the length of so many parts of other tiles
    long long vec, slots, bytes;
};

BwdPlan bwd_plan(int B, int Hq, int Hkv, int Nq, int Nkv, int d, int window, int sinks) {
    BwdPlan p;
    p.window = window < Nkv ? window : Nkv;
    p.sinks = sinks < Nkv ? sinks : Nkv;
    p.nk = (Nkv + 127) / 128;
    p.ns = (p.sinks + 127) / 128;
    p.n_pad = (Nq + 127) / 128 * 128;
    const int nt = bfk::winb::NT;
    const long long units = (long long)B * Hkv, group = Hq / Hkv;
    // Steps of a tile that only its window's queries see, and of one that holds sinks.
    const long long seen = (long long)p.window + 127 < Nq ? (long long)p.window + 127 : Nq;
    const long long norm = group * ((seen + nt - 1) / nt), sink = group * ((Nq + nt - 1) / nt);
    const long long total = units * ((p.nk - p.ns) * norm + p.ns * sink);
    // Two items a multiprocessor where the work allows it, none shorter than 16 steps (below
    // that a part's own fp32 output weighs more than what it reads). A sink tile stays whole
    // where it is no longer than a multiprocessor's mean (in parts of 64 steps: 1 to 8 % slower,
    // the join's time and launch). A longer one comes in parts of about the other items'
    // length, in all at most eight parts a multiprocessor beside whole tiles (that bounds the
    // workspace: 1184 parts are 155 MB at d = 128).
    long long target = (total + 2 * kPlanSms - 1) / (2 * kPlanSms);
    if (target < 16) target = 16;
    p.splits_n = norm * 2 > target * 3 ? (int)((norm + target - 1) / target) : 1;
    const long long floor_s = target < 64 ? target : 64;
    long long target_s = p.splits_n > 1 ? target : (norm > floor_s ? norm : floor_s);
    const long long least = (units * p.ns * sink + 8 * kPlanSms - 1) / (8 * kPlanSms);
    if (target_s < least) target_s = least;
    if (p.splits_n == 1 && sink * kPlanSms <= total) target_s = sink;
    p.splits_s = sink * 2 > target_s * 3 ? (int)((sink + target_s - 1) / target_s) : 1;
    const long long len_s = sink / p.splits_s, len_n = norm / p.splits_n;
    p.times = (int)((len_s + len_n / 2) / (len_n > 0 ? len_n : 1));
    p.vec = (long long)B * Hq * p.n_pad;
    p.slots = units * ((p.splits_s > 1 ? (long long)p.ns * p.splits_s : 0) +
                       (p.splits_n > 1 ? (long long)(p.nk - p.ns) * p.splits_n : 0));
    p.bytes = 4 * (6 * p.vec + p.slots * 2 * 128 * d);
    return p;
}

// The sizes of the backward and its plan. The limits of a launch come before the plan: within
// them its products fit 64 bits.
int check_bwd(int B, int Hq, int Hkv, int Nq, int Nkv, int d, int window, int sinks, float scale, BwdPlan* plan) {
    int rc;
    if ((rc = check_window(B, Hq, Hkv, Nq, Nkv, d, window, sinks, scale)) != BF_OK) return rc;
    const long long heads = (long long)B * Hq, n_pad = (Nq + 127) / 128 * 128;
    bool fits = heads <= 0x7fffffffLL && heads * n_pad / 8 <= 0x7fffffffLL &&
                (Hq / Hkv) * (n_pad / bfk::winb::NT) <= 0x7fffffffLL;
    if (fits) {
        *plan = bwd_plan(B, Hq, Hkv, Nq, Nkv, d, window, sinks);
        const long long parts = (long long)plan->ns * plan->splits_s + (long long)(plan->nk - plan->ns) * plan->splits_n;
        fits = parts <= 0x7fffffffLL / ((long long)B * Hkv);
    }
    return fits ? BF_OK : bf_set_error(BF_ERR_ARG, "problem too large for one launch");
}

// `first`: dK/dV items of sink tiles, which come first, and how many times the others' length they
// have. Blocks that begin with one of them take so many items less of the others: with all in
// turn, 32 blocks at B=2 H=16 N=4096 window 1024 had 172 steps where the mean is 134 (the
// backward there, d = 64: 240 -> 224 us; d = 128 window 512: 226 -> 203).
struct FirstItems {
    long long count;
    int times;
};

template <int D, bool kDQ>
int launch_bwd(const CUtensorMap& x0, const CUtensorMap& x1, const CUtensorMap& y0, const CUtensorMap& y1,
               bfk::winb::Params p, FirstItems first, cudaStream_t stream) {
    static std::atomic<bool> done[64];  // per device; zero-initialised (static storage)
    auto kernel = bfk::winb::window_bwd_kernel<D, kDQ>;
    int rc, sms = 0;
    if ((rc = allow_smem(kernel, bfk::winb::smem_bytes<D, kDQ>(), done)) != BF_OK) return rc;
    if ((rc = sm_count(&sms)) != BF_OK) return rc;
    const int grid = p.items < sms ? p.items : sms;  // persistent: one block per multiprocessor
    p.places = p.late_from = p.items;
    const int late = (int)(first.count % grid);
    if (late > 0 && first.times > 1) {
        // The row of the list in which `late` blocks still have a first item gives the others one
        // item; after it come times - 1 rows for them alone, while there are items.
        const long long from = first.count - late + grid, rest = p.items - from;
        const long long rows = rest > 0 ? (rest + grid - late - 1) / (grid - late) : 0;
        const long long late_rows = rows < first.times - 1 ? rows : first.times - 1;
        if (p.items + late_rows * late <= 0x7fffffffLL - grid) {
            p.late_from = (int)(from < p.items ? from : p.items);
            p.late_rows = (int)late_rows;
            p.late_blocks = late;
            p.places = (int)(p.items + late_rows * late);
        }
    }
    return launch_error(launch_pdl(kernel, dim3((unsigned)grid), bfk::winb::kThreads, bfk::winb::smem_bytes<D, kDQ>(),
                                   stream, x0, x1, y0, y1, p));
}

}  // namespace

extern "C" long long blackflash_window_bwd_workspace_bytes(int B, int Hq, int Hkv, int Nq, int Nkv, int d, int window,
                                                           int sinks) {
    bf_set_error(BF_OK, "");
    BwdPlan plan;
    return check_bwd(B, Hq, Hkv, Nq, Nkv, d, window, sinks, 1.f, &plan) == BF_OK ? plan.bytes : -1;
}

extern "C" int blackflash_window_bwd(const bf_view* Q, const bf_view* K, const bf_view* V, const void* O, const bf_view* dO,
                                     const float* lse, void* dQ, void* dK, void* dV, void* workspace,
                                     long long workspace_bytes, int B, int Hq, int Hkv, int Nq, int Nkv, int d, int window,
                                     int sinks, float scale, void* stream) {
    bf_set_error(BF_OK, "");
    int rc;
    BwdPlan plan;
    if ((rc = check_bwd(B, Hq, Hkv, Nq, Nkv, d, window, sinks, scale, &plan)) != BF_OK) return rc;
    ViewStrides sq, sk, sv, sd;
    if ((rc = check_view(Q, "Q", B, Hq, Nq, d, 2, &sq)) != BF_OK) return rc;
    if ((rc = check_view(K, "K", B, Hkv, Nkv, d, 2, &sk)) != BF_OK) return rc;
    if ((rc = check_view(V, "V", B, Hkv, Nkv, d, 2, &sv)) != BF_OK) return rc;
    if ((rc = check_view(dO, "dO", B, Hq, Nq, d, 2, &sd)) != BF_OK) return rc;
    const void* ptrs[] = {O, dQ, dK, dV, workspace};
    for (const void* ptr : ptrs)
        if (!ptr || (reinterpret_cast<uintptr_t>(ptr) & 31u))
            return bf_set_error(BF_ERR_ARG, "O, dQ, dK, dV and the workspace must be non-null and 32-byte aligned");
    if (!lse) return bf_set_error(BF_ERR_ARG, "lse: null pointer");
    if (workspace_bytes < plan.bytes)
        return bf_set_error(BF_ERR_ARG, "workspace smaller than blackflash_window_bwd_workspace_bytes()");
    const int nt = bfk::winb::NT;
    const int q_tiles = plan.n_pad / 128;
    const long long units = (long long)B * Hkv;
    const long long kv_items = units * ((long long)plan.ns * plan.splits_s + (long long)(plan.nk - plan.ns) * plan.splits_n);
    const long long q_items = (long long)B * Hq * q_tiles;

    if ((rc = bind_context()) != BF_OK) return rc;
    cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
    float* nlse2 = reinterpret_cast<float*>(workspace);
    float* nd = nlse2 + plan.vec;
    uint4* aug = reinterpret_cast<uint4*>(nd + plan.vec);  // vec is a multiple of 128: 16-byte aligned
    float* part = reinterpret_cast<float*>(aug + plan.vec);
    {
        const int per = 256 / (d / 8) * bfk::winb::kPrepRows;  // rows of a block: divides 128
        const int chunks = plan.n_pad / per;
        const dim3 grid((unsigned)(B * Hq), (unsigned)(chunks < 65535 ? chunks : 65535));
        const bool all_swept = plan.window <= bfk::winb::kFewKeys - plan.sinks;  // D comes from the dQ pass
        auto kernel = d == 64 ? bfk::winb::prep_kernel<64> : bfk::winb::prep_kernel<128>;
        if ((rc = launch_error(launch_pdl(kernel, grid, 256, 0, st, reinterpret_cast<const __nv_bfloat16*>(O),
                                          reinterpret_cast<const char*>(dO->data), sd.s[0] * 2, sd.s[1] * 2, sd.s[2] * 2, lse,
                                          nlse2, nd, aug, 1.f / scale, Hq, Nq, plan.n_pad, all_swept ? 0 : 1))) != BF_OK)
            return rc;
    }
    const long long dq[4] = {d, Nq, Hq, B}, dk[4] = {d, Nkv, Hkv, B};
    const long long tq[3] = {sq.s[2], sq.s[1], sq.s[0]}, tk[3] = {sk.s[2], sk.s[1], sk.s[0]},
                    tv[3] = {sv.s[2], sv.s[1], sv.s[0]}, td[3] = {sd.s[2], sd.s[1], sd.s[0]};
    // Stationary tiles in 128-row boxes [0], streamed ones in nt-row boxes [1].
    CUtensorMap mq[2], mk[2], mv[2], md[2];
    for (int i = 0; i < 2; ++i) {
        const int box = i ? nt : 128;
        if ((rc = make_map_4d(&mq[i], Q->data, false, dq, tq, box, 1)) != BF_OK) return rc;
        if ((rc = make_map_4d(&md[i], dO->data, false, dq, td, box, 1)) != BF_OK) return rc;
        if ((rc = make_map_4d(&mk[i], K->data, false, dk, tk, box, 1)) != BF_OK) return rc;
        if ((rc = make_map_4d(&mv[i], V->data, false, dk, tv, box, 1)) != BF_OK) return rc;
    }

    bfk::winb::Params p;
    memset(&p, 0, sizeof(p));
    p.batch = B;
    p.hq = Hq;
    p.hkv = Hkv;
    p.group = Hq / Hkv;
    p.n_q = Nq;
    p.n_kv = Nkv;
    p.n_pad = plan.n_pad;
    p.nk = plan.nk;
    p.ns = plan.ns;
    p.window = plan.window;
    p.sinks = plan.sinks;
    p.q_tiles = q_tiles;
    p.splits_s = plan.splits_s;
    p.splits_n = plan.splits_n;
    p.scale = scale;
    p.scale_log2 = scale * kLog2e;
    p.nlse2 = nlse2;
    p.nd = nd;
    p.aug = aug;
    p.dq = reinterpret_cast<__nv_bfloat16*>(dQ);
    p.dk = reinterpret_cast<__nv_bfloat16*>(dK);
    p.dv = reinterpret_cast<__nv_bfloat16*>(dV);
    p.part = part;
    p.timeout_ns = kTimeoutNs;
    p.items = (int)q_items;  // first: it leaves a better D of rows that see few keys
    rc = d == 64 ? launch_bwd<64, true>(mq[0], md[0], mk[1], mv[1], p, {0, 0}, st)
                 : launch_bwd<128, true>(mq[0], md[0], mk[1], mv[1], p, {0, 0}, st);
    if (rc != BF_OK) return rc;
    p.items = (int)kv_items;
    const FirstItems first{units * plan.ns * plan.splits_s, plan.times};
    rc = d == 64 ? launch_bwd<64, false>(mk[0], mv[0], mq[1], md[1], p, first, st)
                 : launch_bwd<128, false>(mk[0], mv[0], mq[1], md[1], p, first, st);
    if (rc != BF_OK) return rc;
    auto join = [&](const float* from, int j0, int tiles, int splits) -> int {
        if (splits <= 1 || tiles <= 0) return BF_OK;
        const long long threads = units * tiles * 2 * 128 * (d / 4);
        if (threads / 256 >= 0x7fffffffLL) return bf_set_error(BF_ERR_ARG, "problem too large for one launch");
        auto kernel = d == 64 ? bfk::winb::join_kernel<64> : bfk::winb::join_kernel<128>;
        return launch_error(launch_pdl(kernel, dim3((unsigned)((threads + 255) / 256)), 256, 0, st, from, p.dk, p.dv, j0, tiles,
                                       splits, Nkv, units));
    };
    if ((rc = join(part, 0, plan.ns, plan.splits_s)) != BF_OK) return rc;
    const float* rest = part + (plan.splits_s > 1 ? units * plan.ns * plan.splits_s * 2 * 128 * d : 0);
    return join(rest, plan.ns, plan.nk - plan.ns, plan.splits_n);
}

int bf_prefix_partial(const PrefixArgs& a) {
    int rc;
    ViewStrides sk, sv;
    if ((rc = check_view(&a.k, "K_prefix", 1, a.Hkv, a.P, a.d, 2, &sk)) != BF_OK) return rc;
    if ((rc = check_view(&a.v, "V_prefix", 1, a.Hkv, a.P, a.d, 2, &sv)) != BF_OK) return rc;
    bfk::win::Params p;
    memset(&p, 0, sizeof(p));
    p.batch = a.B;
    p.hq = a.Hq;
    p.hkv = a.Hkv;
    p.group = a.Hq / a.Hkv;
    p.n_q = a.T;
    p.n_kv = a.P;
    p.nk = (a.P + 127) / 128;
    p.scale_log2 = a.scale * kLog2e;
    p.out = a.o;
    p.lse = a.lse2;
    p.timeout_ns = kTimeoutNs;
    p.q_rows = p.group * a.T;
    p.seqs_per_tile = 128 / p.q_rows;  // 0: a sequence's rows span several tiles
    p.tiles_per_seq = (p.q_rows + 127) / 128;
    p.row_tiles = p.seqs_per_tile ? (a.B + p.seqs_per_tile - 1) / p.seqs_per_tile : a.B * p.tiles_per_seq;
    p.pairs = (p.row_tiles + 1) / 2;
    p.split_tiles = a.split_tiles;
    p.rows = (long long)a.B * a.Hq * a.T;
    const long long items = (long long)p.pairs * a.Hkv * a.splits;
    if (items > 0x7fffffffLL) return bf_set_error(BF_ERR_ARG, "problem too large for one launch");
    p.items = (int)items;

    CUtensorMap mq, mk, mv;
    const long long dq[4] = {a.d, p.q_rows, a.B, a.Hkv}, dk[4] = {a.d, a.P, a.Hkv, 1};
    const long long tq[3] = {a.d, (long long)a.Hkv * p.q_rows * a.d, (long long)p.q_rows * a.d};
    const long long tk[3] = {sk.s[2], sk.s[1], sk.s[0]}, tv[3] = {sv.s[2], sv.s[1], sv.s[0]};
    if ((rc = make_map_4d(&mq, a.q, a.f16, dq, tq, p.seqs_per_tile ? p.q_rows : 128,
                          p.seqs_per_tile ? p.seqs_per_tile : 1)) != BF_OK)
        return rc;
    if ((rc = make_map_4d(&mk, a.k.data, a.f16, dk, tk, 128, 1)) != BF_OK) return rc;
    if ((rc = make_map_4d(&mv, a.v.data, a.f16, dk, tv, 128, 1)) != BF_OK) return rc;
    return launch_fwd<true, false>(a.d, a.f16, mq, mk, mv, p, a.stream);
}

int bf_window_wait_status(int reset, unsigned* out) {
    cudaError_t e = cudaMemcpyFromSymbol(out, bfk::g_wait_status, sizeof(*out));
    if (e == cudaSuccess && reset) {
        const unsigned zero = 0;
        e = cudaMemcpyToSymbol(bfk::g_wait_status, &zero, sizeof(zero));
    }
    return e == cudaSuccess ? BF_OK : bf_set_error(BF_ERR_CUDA, cudaGetErrorString(e));
}
