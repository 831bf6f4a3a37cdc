// Rotary positions: pair i of a token at position n is turned by the angle n * freq[i] and
// stretched by an amplitude,
//   (u, w) -> a (u cos - w sin, u sin + w cos),
// for Q and K in one launch. Pairs are neighbours (interleaved) or the two halves of the
// rotated part; the columns past it are copied. The gradient is the same map with the
// angle's sign turned.
//
// Bound by memory: every element is read once and written once. The angle needs 64 bits,
// because at position 10^6 a 32-bit product is off by 0.06 rad: it is formed in turns
// (freq / 2 pi, in fp64), reduced to [-1/2, 1/2] there, and only then taken to fp32 and
// sincospi. A block does this once for its tokens and all of their heads, into shared
// memory, so the fp64 work is one product and one rounding per (token, pair).
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <math.h>
#include <string.h>

#include "sm100_ptx.cuh"
#include "views.h"

namespace bfk {
namespace rot {

struct Params {
    const char* x[2];       // Q, K (null: absent)
    char* y[2];             // contiguous [B, H, N, d]
    long long xs[2][3];     // byte strides of batch, head, token
    int heads[2];
    const void* positions;  // [N] or [B, N], int32 or int64
    long long pos_stride;   // 0 or N
    const double* freqs;    // [rot / 2], radians per position
    float amplitude, sign;
    long long tokens;       // B * N
    int n, d, rot, pos64;
    int tile;               // tokens of a block
    int head_split;         // blocks along the heads
};

template <typename T>
__device__ __forceinline__ float to_f(T v);
template <>
__device__ __forceinline__ float to_f<float>(float v) { return v; }
template <>
__device__ __forceinline__ float to_f<__nv_bfloat16>(__nv_bfloat16 v) { return __bfloat162float(v); }
template <>
__device__ __forceinline__ float to_f<__half>(__half v) { return __half2float(v); }
template <typename T>
__device__ __forceinline__ T from_f(float v);
template <>
__device__ __forceinline__ float from_f<float>(float v) { return v; }
template <>
__device__ __forceinline__ __nv_bfloat16 from_f<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }
template <>
__device__ __forceinline__ __half from_f<__half>(float v) { return __float2half_rn(v); }

// The turn, its fused products written out: left to the compiler, they were fused the one way or
// the other by vector width, and a view's alignment showed in the last bit.
__device__ __forceinline__ float turn_u(float u, float w, float2 cs) { return fmaf(u, cs.x, -__fmul_rn(w, cs.y)); }
__device__ __forceinline__ float turn_w(float u, float w, float2 cs) { return fmaf(u, cs.y, __fmul_rn(w, cs.x)); }

template <typename T, int V>
struct __align__(sizeof(T) * V) Vec {
    T e[V];
};

constexpr int kBlock = 256;
constexpr int kMaxTile = 4;      // tokens of a block: 72 us at B=4 N=4095 Hq=32 Hk=8 d=128 (a copy: 58), 8: 74, 2: 75
constexpr int kMaxPairs = 512;  // (token, pair) entries of a block's table

// A work item is V consecutive columns of one row: of the first half with their partners of
// the second half (half layout), of the rotated part (interleaved), or copied columns. A thread
// keeps its item and steps through the rows (token, head) of its block. Few registers and a
// full multiprocessor of threads (2048) carry more bytes in flight than more loads a thread do.
template <typename T, int V, bool kInterleaved>
__global__ void __launch_bounds__(kBlock, 8) rotary_kernel(const Params p) {
    __shared__ float2 cs[kMaxPairs];
    __shared__ const char* x_at[2][kMaxTile];  // a token's row of head 0
    __shared__ char* y_at[2][kMaxTile];
    __shared__ long long pos_at[kMaxTile];
    const int half = p.rot / 2;
    const long long t0 = (long long)blockIdx.x * p.tile;
    const int nt = (int)min((long long)p.tile, p.tokens - t0);
    griddep_launch_dependents();
    griddep_wait();
    if (threadIdx.x < nt) {
        const long long tok = t0 + threadIdx.x, b = tok / p.n, n = tok - b * p.n;
#pragma unroll
        for (int w = 0; w < 2; ++w) {
            x_at[w][threadIdx.x] = p.x[w] + b * p.xs[w][0] + n * p.xs[w][2];
            y_at[w][threadIdx.x] = p.y[w] + (b * p.heads[w] * p.n + n) * p.d * (int)sizeof(T);
        }
        pos_at[threadIdx.x] = b * p.pos_stride + n;
    }
    __syncthreads();

    for (int i = threadIdx.x; i < nt * half; i += kBlock) {
        const int tt = i / half, pr = i - tt * half;
        const long long at = pos_at[tt];
        const long long pos = p.pos64 ? reinterpret_cast<const long long*>(p.positions)[at]
                                      : (long long)reinterpret_cast<const int*>(p.positions)[at];
        const double turns = (double)pos * (p.freqs[pr] * 0.15915494309189533577);
        const double angle = 2.0 * (turns - rint(turns));  // in units of pi, [-1, 1]
        const float hi = (float)angle;
        float s, co;
        sincospif(hi, &s, &co);
        // First-order step for what the cast to fp32 dropped (up to 2^-24 of the angle).
        const float lo = (float)(angle - (double)hi) * 3.14159265f;
        cs[i] = make_float2(fmaf(-s, lo, co) * p.amplitude, fmaf(co, lo, s) * p.amplitude * p.sign);
    }
    __syncthreads();

    const int rot_items = kInterleaved ? p.rot / V : half / V;  // of a row; then the copied ones
    const int row_items = rot_items + (p.d - p.rot) / V;
    const int all_heads = p.heads[0] + p.heads[1];
    const int h0 = (int)((long long)all_heads * blockIdx.y / p.head_split);
    const int nh = (int)((long long)all_heads * (blockIdx.y + 1) / p.head_split) - h0;
    const int across = min(row_items, kBlock), pass = kBlock / across;  // rows of a pass
    const int first = threadIdx.x / across;
    if (first >= pass) return;
    using VT = Vec<T, V>;
    const long long y_head = (long long)p.n * p.d * (int)sizeof(T);
    for (int item = threadIdx.x - first * across; item < row_items; item += kBlock) {
        const bool turned = item < rot_items;
        const int col = turned ? item * V : p.rot + (item - rot_items) * V;
        int t = first / nh, h = first - t * nh;
        while (t < nt) {
            const int hh = h0 + h, w = hh >= p.heads[0], hw = w ? hh - p.heads[0] : hh;
            const T* x = reinterpret_cast<const T*>(x_at[w][t] + hw * p.xs[w][1]) + col;
            T* y = reinterpret_cast<T*>(y_at[w][t] + hw * y_head) + col;
            VT a = *reinterpret_cast<const VT*>(x);
            if (turned) {
                const float2* tab = cs + t * half + (kInterleaved ? col >> 1 : col);
                if constexpr (kInterleaved) {
#pragma unroll
                    for (int e = 0; e < V; e += 2) {
                        const float2 cw = tab[e >> 1];
                        const float u = to_f<T>(a.e[e]), v = to_f<T>(a.e[e + 1]);
                        a.e[e] = from_f<T>(turn_u(u, v, cw));
                        a.e[e + 1] = from_f<T>(turn_w(u, v, cw));
                    }
                } else {
                    VT c = *reinterpret_cast<const VT*>(x + half);
#pragma unroll
                    for (int e = 0; e < V; ++e) {
                        const float2 cw = tab[e];
                        const float u = to_f<T>(a.e[e]), v = to_f<T>(c.e[e]);
                        a.e[e] = from_f<T>(turn_u(u, v, cw));
                        c.e[e] = from_f<T>(turn_w(u, v, cw));
                    }
                    *reinterpret_cast<VT*>(y + half) = c;
                }
            }
            *reinterpret_cast<VT*>(y) = a;
            h += pass;
            while (h >= nh) {
                h -= nh;
                ++t;
            }
        }
    }
}

template <typename T, int V, bool kInterleaved>
int launch(const Params& p, dim3 grid, cudaStream_t stream) {
    return launch_error(launch_pdl(rotary_kernel<T, V, kInterleaved>, grid, kBlock, 0, stream, p));
}

// V = 16 bytes where every piece of a row, its start and its strides are whole 16-byte vectors,
// else a pair for the interleaved layout and one column for halves. bf16, B=4 N=4095 Hq=32 Hk=8
// d=80, where a copy takes 42 us: 46 to 48 us with 32 or 80 columns turned; with 20 turned a pair 83
// and one column 130 us, with 40 (whose halves are 20) 119. Vectors between are not built.
template <typename T>
int launch_v(const Params& p, int v, bool interleaved, dim3 grid, cudaStream_t stream) {
    constexpr int kMax = 16 / (int)sizeof(T);
    if (interleaved) {
        if (v == kMax) return launch<T, kMax, true>(p, grid, stream);
        return launch<T, 2, true>(p, grid, stream);
    }
    if (v == kMax) return launch<T, kMax, false>(p, grid, stream);
    return launch<T, 1, false>(p, grid, stream);
}

}  // namespace rot
}  // namespace bfk

extern "C" int blackflash_rotary(const bf_view* Q, const bf_view* K, void* Q_out, void* K_out, const void* positions,
                                 int positions_64, int positions_per_batch, const double* freqs, int B, int Hq, int Hk,
                                 int N, int d, int rotary_dim, int interleaved, float amplitude, int inverse, int dtype,
                                 void* stream) {
    bf_set_error(BF_OK, "");
    if (B <= 0 || N <= 0 || Hq < 0 || Hk < 0 || Hq + Hk <= 0)
        return bf_set_error(BF_ERR_ARG, "empty problem: B, N and the heads must be >= 1");
    if (Hq > 65536 || Hk > 65536) return bf_set_error(BF_ERR_ARG, "more than 65536 heads");
    if (d <= 0 || d > 1024 || d % 2 || rotary_dim < 2 || rotary_dim > d || rotary_dim % 2)
        return bf_set_error(BF_ERR_ARG, "need an even d <= 1024 and an even rotary_dim in [2, d]");
    if (!positions || !freqs) return bf_set_error(BF_ERR_ARG, "null pointer");
    if (!isfinite(amplitude)) return bf_set_error(BF_ERR_ARG, "amplitude must be finite");
    if (dtype != BF_DTYPE_BF16 && dtype != BF_DTYPE_F16 && dtype != BF_DTYPE_F32)
        return bf_set_error(BF_ERR_ARG, "dtype must be bf16, fp16 or fp32");
    const int size = dtype == BF_DTYPE_F32 ? 4 : 2;
    bfk::rot::Params p;
    memset(&p, 0, sizeof(p));
    const bf_view* in[2] = {Q, K};
    void* out[2] = {Q_out, K_out};
    const int heads[2] = {Hq, Hk};
    const int full = 16 / size;
    // Every boundary inside a row, and every row's start, on whole vectors?
    bool vec = d % full == 0 && rotary_dim % full == 0 && (interleaved || rotary_dim / 2 % full == 0);
    for (int i = 0; i < 2; ++i) {
        p.heads[i] = heads[i];
        if (!heads[i]) continue;
        if (!in[i] || !in[i]->data || !out[i]) return bf_set_error(BF_ERR_ARG, "null pointer");
        const uintptr_t at = reinterpret_cast<uintptr_t>(in[i]->data), to = reinterpret_cast<uintptr_t>(out[i]);
        if (at % (2 * size) || to % (2 * size)) return bf_set_error(BF_ERR_ARG, "Q and K must start on whole pairs");
        vec = vec && at % 16 == 0 && to % 16 == 0;
        p.x[i] = reinterpret_cast<const char*>(in[i]->data);
        p.y[i] = reinterpret_cast<char*>(out[i]);
        const int n[3] = {B, heads[i], N};
        for (int k = 0; k < 3; ++k) {
            const long long s = n[k] > 1 ? in[i]->stride[k] : 0;
            if (s < 0 || s % 2) return bf_set_error(BF_ERR_ARG, "strides must be even and not negative");
            vec = vec && s % full == 0;
            p.xs[i][k] = s * size;
        }
    }
    const int v = vec ? full : (interleaved ? 2 : 1);
    p.positions = positions;
    p.pos64 = positions_64 != 0;
    p.pos_stride = positions_per_batch ? N : 0;
    p.freqs = freqs;
    p.amplitude = amplitude;
    p.sign = inverse ? -1.f : 1.f;
    p.tokens = (long long)B * N;
    p.n = N;
    p.d = d;
    p.rot = rotary_dim;
    // Tokens of a block: enough that one pass of its threads fills the table, fewer where that
    // would leave multiprocessors without a block; then the heads are split too.
    int tile = bfk::rot::kBlock / (rotary_dim / 2);
    if (tile < 1) tile = 1;
    if (tile > bfk::rot::kMaxTile) tile = bfk::rot::kMaxTile;
    const long long even = (p.tokens + 2 * kPlanSms - 1) / (2 * kPlanSms);
    if (even < tile) tile = (int)even;
    p.tile = tile;
    const long long blocks = (p.tokens + tile - 1) / tile;
    if (blocks > 0x7fffffffLL) return bf_set_error(BF_ERR_ARG, "problem too large for one launch");
    long long hs = (2 * kPlanSms + blocks - 1) / blocks;
    if (hs > Hq + Hk) hs = Hq + Hk;
    if (hs > 65535) hs = 65535;
    p.head_split = (int)hs;
    const dim3 grid((unsigned)blocks, (unsigned)hs);
    cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
    if (dtype == BF_DTYPE_F32) return bfk::rot::launch_v<float>(p, v, interleaved != 0, grid, st);
    if (dtype == BF_DTYPE_F16) return bfk::rot::launch_v<__half>(p, v, interleaved != 0, grid, st);
    return bfk::rot::launch_v<__nv_bfloat16>(p, v, interleaved != 0, grid, st);
}
