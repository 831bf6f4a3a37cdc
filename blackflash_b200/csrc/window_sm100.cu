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

}  // namespace bfk

namespace {

constexpr unsigned long long kTimeoutNs = 4000000000ull;
constexpr float kLog2e = 1.4426950408889634f;

template <int D, bool kF16, bool kPartial>
int launch_fwd(const CUtensorMap& mq, const CUtensorMap& mk, const CUtensorMap& mv, const bfk::win::Params& p,
               cudaStream_t stream) {
    static std::atomic<bool> done[64];  // per device; zero-initialised (static storage)
    auto kernel = bfk::win::window_fwd_kernel<D, kF16, kPartial>;
    int rc, sms = 0;
    if ((rc = allow_smem(kernel, bfk::win::smem_bytes<D>(), done)) != BF_OK) return rc;
    if ((rc = sm_count(&sms)) != BF_OK) return rc;
    const int grid = p.items < sms ? p.items : sms;  // persistent: at most one CTA per SM
    return launch_error(launch_pdl(kernel, dim3((unsigned)grid), bfk::win::kThreads, bfk::win::smem_bytes<D>(), stream, mq,
                                   mk, mv, p));
}

template <bool kPartial>
int launch_fwd(int d, bool f16, const CUtensorMap& mq, const CUtensorMap& mk, const CUtensorMap& mv,
               const bfk::win::Params& p, cudaStream_t stream) {
    if (d == 64)
        return f16 ? launch_fwd<64, true, kPartial>(mq, mk, mv, p, stream)
                   : launch_fwd<64, false, kPartial>(mq, mk, mv, p, stream);
    return f16 ? launch_fwd<128, true, kPartial>(mq, mk, mv, p, stream)
               : launch_fwd<128, false, kPartial>(mq, mk, mv, p, stream);
}

int check_window(int B, int Hq, int Hkv, int Nq, int Nkv, int d, int window, int sinks, float scale) {
    if (B <= 0 || Hq <= 0 || Hkv <= 0 || Nq <= 0 || Nkv <= 0)
        return bf_set_error(BF_ERR_ARG, "empty problem: B, H and N must be >= 1");
    if (Hq % Hkv) return bf_set_error(BF_ERR_ARG, "query heads must be a multiple of KV heads");
    if (d != 64 && d != 128) return bf_set_error(BF_ERR_ARG, "BlackFlash supports d=64 and d=128");
    if (Nq > (1 << 30) || Nkv > (1 << 30)) return bf_set_error(BF_ERR_ARG, "more than 2^30 rows");
    if (window < 1 || sinks < 0) return bf_set_error(BF_ERR_ARG, "need window >= 1 and sinks >= 0");
    if (!(scale > 0.f) || !isfinite(scale)) return bf_set_error(BF_ERR_ARG, "scale must be positive and finite");
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
    if (!O || (reinterpret_cast<uintptr_t>(O) & 15u)) return bf_set_error(BF_ERR_ARG, "O must be 16-byte aligned");

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

    if ((rc = bind_context()) != BF_OK) return rc;
    const bool f16 = dtype == BF_DTYPE_F16;
    CUtensorMap mq, mk, mv;
    const long long dq[4] = {d, Nq, Hq, B}, dk[4] = {d, Nkv, Hkv, B};
    const long long tq[3] = {sq.s[2], sq.s[1], sq.s[0]}, tk[3] = {sk.s[2], sk.s[1], sk.s[0]},
                    tv[3] = {sv.s[2], sv.s[1], sv.s[0]};
    if ((rc = make_map_4d(&mq, Q->data, f16, dq, tq, 128, 1)) != BF_OK) return rc;
    if ((rc = make_map_4d(&mk, K->data, f16, dk, tk, 128, 1)) != BF_OK) return rc;
    if ((rc = make_map_4d(&mv, V->data, f16, dk, tv, 128, 1)) != BF_OK) return rc;
    return launch_fwd<false>(d, f16, mq, mk, mv, p, reinterpret_cast<cudaStream_t>(stream));
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
    return launch_fwd<true>(a.d, a.f16, mq, mk, mv, p, a.stream);
}

int bf_window_wait_status(int reset, unsigned* out) {
    cudaError_t e = cudaMemcpyFromSymbol(out, bfk::g_wait_status, sizeof(*out));
    if (e == cudaSuccess && reset) {
        const unsigned zero = 0;
        e = cudaMemcpyToSymbol(bfk::g_wait_status, &zero, sizeof(zero));
    }
    return e == cudaSuccess ? BF_OK : bf_set_error(BF_ERR_CUDA, cudaGetErrorString(e));
}
