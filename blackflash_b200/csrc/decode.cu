// Decoding steps: one or a few new tokens of each sequence against its cache, with a
// sliding window and sinks, or behind a prefix that the whole batch shares.
//
// A step reads every visible key and value once and computes 2 * rows products per element
// read, rows = group * T (query heads of a KV head times new tokens): far below the
// 250 operations a byte at which the tensor core would bound it, so the kernel is built
// for bytes in flight. A block is four warps (eight where it takes few keys and has a
// multiprocessor to itself) that share nothing but the last join: each walks its own 16-byte
// cp.async pipeline over groups of keys, multiplies them with all 16 rows of the tile by
// m16n8k16, and keeps its own running maximum, sum and output. Keys
// past a sequence's length are filled with zeros in shared memory and never read from
// memory, so what a cache holds there (infinities, NaN, addresses past its end) does not
// matter. The visible keys of a row tile are [0, s0) and [lo, hi); they are numbered
// through, so that sinks cost no extra pass (nor a short shared prefix, whose keys then come
// first), and split into chunks over blocks. Chunks
// leave fp32 partials and their log2-sum-exp2, joined by combine_kernel.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <math.h>
#include <string.h>

#include "sm100_ptx.cuh"
#include "views.h"

namespace bfk {
namespace dec {

constexpr int kWarps = 4;      // of a block
constexpr int kWideWarps = 8;  // of a block that has a multiprocessor to itself (Plan::wide)
constexpr int kStages = 2;  // 64 KiB a block, three blocks a multiprocessor; three stages and two blocks: 3 to 10 % slower

template <int D, int W>
struct Cfg {
    static constexpr int kKeys = 2048 / D;          // keys of a warp's step: 4 KiB each of K and V
    static constexpr int kRow = D * 2;              // bytes of a row
    static constexpr int kChunks = kRow / 16;       // 16-byte chunks of a row
    static constexpr int kHalf = kKeys * kRow;      // K (or V) bytes of a stage
    static constexpr int kStage = 2 * kHalf;
    static constexpr int kWarpBytes = kStages * kStage;
    static constexpr int kSmem = W * kWarpBytes;
    static_assert(kWarpBytes >= 16 * (D + 4) * 4, "the join reuses a warp's stages");
};

struct Params {
    const void* q;      // [B, Hq, T, D]
    const char* k;
    const char* v;
    long long ks[3], vs[3];  // byte strides of batch, head, token
    const int* lengths;
    void* out;          // direct: [B, Hq, T, D] bf16 / fp16
    float* lse;         // direct: [B, Hq, T] natural log, optional
    float* part_o;      // split: [splits][rows][D], null for direct
    float* part_lse;    // split: [splits][rows] log2
    long long rows;     // B * Hq * T
    int hkv, q_rows, tokens, cap, row_tiles;
    int window, sinks;  // clamped to cap
    int chunk;          // keys of a split
    const char *kp, *vp;          // kPrefix: the shared prefix, whose keys come before the cache's
    long long kps[2], vps[2];     // byte strides of head, token
    int prefix;
    int beside;         // the grid before is the prefix part: do not wait for it at the start
    float scale_log2;
};

__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src, bool valid) {
    const int n = valid ? 16 : 0;  // 0: sixteen zero bytes, nothing read
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(n) : "memory");
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_async_wait() {
    asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}
__device__ __forceinline__ void ldsm4(uint32_t addr, uint32_t (&r)[4]) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(addr)
                 : "memory");
}
__device__ __forceinline__ void ldsm4_t(uint32_t addr, uint32_t (&r)[4]) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(addr)
                 : "memory");
}
template <bool kF16>
__device__ __forceinline__ void mma16816(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    if constexpr (kF16)
        asm volatile(
            "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
            "{%0, %1, %2, %3};"
            : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
            : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
    else
        asm volatile(
            "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
            "{%0, %1, %2, %3};"
            : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
            : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

template <bool kF16>
__device__ __forceinline__ uint32_t pack2(float lo, float hi) {
    return kF16 ? pack_f16x2(lo, hi) : pack_bf16x2(lo, hi);
}

// kPrefix: the prefix's keys are the first of the numbering, as sinks are, and every token sees
// them; each sequence reads them for itself.
template <int D, bool kF16, bool kPrefix, int W>
__global__ void __launch_bounds__(W * 32) decode_kernel(const Params p) {
    using C = Cfg<D, W>;
    constexpr int NB = C::kKeys / 8;  // score blocks of 8 keys
    extern __shared__ __align__(128) uint8_t smem[];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int split = blockIdx.y;
    const int rt = blockIdx.x % p.row_tiles;
    const int bh = blockIdx.x / p.row_tiles;
    const int kvh = bh % p.hkv, b = bh / p.hkv;
    // Behind the prefix part, this grid was launched only after every grid before that one had
    // completed, and needs nothing of it. But its own completion, for which the join waits,
    // has to mean the prefix part's too: the last block waits for it at its end. The fence keeps
    // the loads of lengths and Q from lines that L1 may still hold from before those grids.
    griddep_launch_dependents();
    if (p.beside)
        __threadfence();
    else
        griddep_wait();

    const int len = kPrefix && p.cap == 0 ? 0 : min(max(p.lengths[b], 0), p.cap);
    const int pos0 = len - p.tokens;  // position of new token 0; may be negative
    const int lo = max(0, pos0 - p.window + 1);
    const int s0 = kPrefix ? p.prefix : min(p.sinks, lo);
    const int n_vis = s0 + len - lo;
    const long long base = (long long)split * p.chunk;
    const int v0 = base < n_vis ? (int)base : n_vis;
    const int v1 = n_vis - v0 < p.chunk ? n_vis : v0 + p.chunk;

    // This thread's two rows of the tile (lane / 4 and + 8), and their positions.
    const int r0 = rt * 16 + (lane >> 2), r1 = r0 + 8;
    const int p0 = pos0 + r0 % p.tokens, p1 = pos0 + r1 % p.tokens;
    const size_t row_base = ((size_t)b * p.hkv + kvh) * p.q_rows;

    uint8_t* mine = smem + warp * C::kWarpBytes;
    const uint32_t mine_a = smem_addr(mine);
    const char* kb = p.k + b * p.ks[0] + kvh * p.ks[1];
    const char* vb = p.v + b * p.vs[0] + kvh * p.vs[1];
    const char* kpb = kPrefix ? p.kp + kvh * p.kps[0] : nullptr;
    const char* vpb = kPrefix ? p.vp + kvh * p.vps[0] : nullptr;
    const int groups = (v1 - v0 + C::kKeys - 1) / C::kKeys;
    const int steps = groups > warp ? (groups - warp + W - 1) / W : 0;

    auto load = [&](int s) {
        if (s < steps) {
            const int vg = v0 + (warp + s * W) * C::kKeys;
            const uint32_t dst = mine_a + (uint32_t)(s % kStages) * C::kStage;
#pragma unroll
            for (int i = 0; i < C::kHalf / 512; ++i) {
                const int row = i * (32 / C::kChunks) + lane / C::kChunks;
                const int ch = lane % C::kChunks;
                const bool valid = vg + row < v1;
                const int v = valid ? vg + row : v0;  // a safe address; nothing is read from it
                const long long key = v < s0 ? v : lo + (v - s0);
                const char *k_row, *v_row;
                if (kPrefix && v < s0) {
                    k_row = kpb + key * p.kps[1];
                    v_row = vpb + key * p.vps[1];
                } else {
                    k_row = kb + key * p.ks[2];
                    v_row = vb + key * p.vs[2];
                }
                const uint32_t at = (uint32_t)row * C::kRow + (uint32_t)((ch ^ (row & 7)) << 4);
                cp_async16(dst + at, k_row + ch * 16, valid);
                cp_async16(dst + C::kHalf + at, v_row + ch * 16, valid);
            }
        }
        cp_async_commit();
    };

    // P is scaled by 2^15 in fp16, where its largest entry is 1: the smallest kept entry is
    // then 2^-39 of it, not 2^-24.
    constexpr float kShift = kF16 ? 15.f : 0.f;
    float m0 = -INFINITY, m1 = -INFINITY, l0 = 0.f, l1 = 0.f;
    float acc[D / 8][4];
#pragma unroll
    for (int i = 0; i < D / 8; ++i)
#pragma unroll
        for (int c = 0; c < 4; ++c) acc[i][c] = 0.f;

#pragma unroll
    for (int s = 0; s < kStages - 1; ++s) load(s);

    // A fragments of Q, requested behind the first keys: rows past the tile's last read as zero.
    uint32_t qf[D / 16][4];
    {
        const uint32_t* q32 = reinterpret_cast<const uint32_t*>(p.q);
        const size_t a0 = (row_base + r0) * (D / 2) + (lane & 3), a1 = (row_base + r1) * (D / 2) + (lane & 3);
#pragma unroll
        for (int kk = 0; kk < D / 16; ++kk) {
            qf[kk][0] = r0 < p.q_rows ? q32[a0 + kk * 8] : 0u;
            qf[kk][1] = r1 < p.q_rows ? q32[a1 + kk * 8] : 0u;
            qf[kk][2] = r0 < p.q_rows ? q32[a0 + kk * 8 + 4] : 0u;
            qf[kk][3] = r1 < p.q_rows ? q32[a1 + kk * 8 + 4] : 0u;
        }
    }

    for (int s = 0; s < steps; ++s) {
        load(s + kStages - 1);
        cp_async_wait<kStages - 1>();
        __syncwarp();
        const uint32_t kst = mine_a + (uint32_t)(s % kStages) * C::kStage, vst = kst + C::kHalf;
        float sc[NB][4];
#pragma unroll
        for (int i = 0; i < NB; ++i)
#pragma unroll
            for (int c = 0; c < 4; ++c) sc[i][c] = 0.f;
#pragma unroll
        for (int kk = 0; kk < D / 16; ++kk) {
#pragma unroll
            for (int i = 0; i < NB / 2; ++i) {
                const int key = i * 16 + ((lane >> 4) << 3) + (lane & 7);
                const int ch = kk * 2 + ((lane >> 3) & 1);
                uint32_t r[4];
                ldsm4(kst + (uint32_t)key * C::kRow + (uint32_t)((ch ^ (key & 7)) << 4), r);
                mma16816<kF16>(sc[2 * i], qf[kk], r[0], r[1]);
                mma16816<kF16>(sc[2 * i + 1], qf[kk], r[2], r[3]);
            }
        }
        // Mask and scale. A group of window keys up to the first token's position and inside the
        // last one's window, or of sinks, is visible to every row.
        const int vg = v0 + (warp + s * W) * C::kKeys;
        const int k0 = lo + (vg - s0), k1 = k0 + C::kKeys - 1;
        const bool whole = vg + C::kKeys <= v1 &&
                           (vg >= s0 ? k1 <= pos0 && len - 1 - k0 < p.window : vg + C::kKeys <= s0);
        float x0 = -INFINITY, x1 = -INFINITY;
#pragma unroll
        for (int i = 0; i < NB; ++i) {
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                float a = sc[i][e] * p.scale_log2, c = sc[i][e + 2] * p.scale_log2;
                if (!whole) {
                    const int v = vg + i * 8 + (lane & 3) * 2 + e;
                    const int key = v < s0 ? v : lo + (v - s0);
                    const bool in = v < v1;
                    const bool sink = kPrefix ? v < s0 : key < p.sinks;
                    const bool before0 = (kPrefix && sink) || key <= p0, before1 = (kPrefix && sink) || key <= p1;
                    if (!(in && before0 && (sink || p0 - key < p.window))) a = -INFINITY;
                    if (!(in && before1 && (sink || p1 - key < p.window))) c = -INFINITY;
                }
                sc[i][e] = a;
                sc[i][e + 2] = c;
                x0 = fmaxf(x0, a);
                x1 = fmaxf(x1, c);
            }
        }
        x0 = fmaxf(x0, __shfl_xor_sync(0xffffffffu, x0, 1));
        x1 = fmaxf(x1, __shfl_xor_sync(0xffffffffu, x1, 1));
        x0 = fmaxf(x0, __shfl_xor_sync(0xffffffffu, x0, 2));
        x1 = fmaxf(x1, __shfl_xor_sync(0xffffffffu, x1, 2));
        const bool up = x0 > m0 || x1 > m1;
        if (__any_sync(0xffffffffu, up)) {
            const float n0 = fmaxf(m0, x0), n1 = fmaxf(m1, x1);
            const float f0 = n0 > m0 ? fast_exp2(m0 - n0) : 1.f, f1 = n1 > m1 ? fast_exp2(m1 - n1) : 1.f;
            m0 = n0;
            m1 = n1;
            l0 *= f0;
            l1 *= f1;
#pragma unroll
            for (int i = 0; i < D / 8; ++i) {
                acc[i][0] *= f0;
                acc[i][1] *= f0;
                acc[i][2] *= f1;
                acc[i][3] *= f1;
            }
        }
        // A row that has seen nothing refers to 0: its masked scores give 2^-inf, not NaN.
        const float b0 = m0 == -INFINITY ? 0.f : kShift - m0, b1 = m1 == -INFINITY ? 0.f : kShift - m1;
        uint32_t pf[NB / 2][4];
#pragma unroll
        for (int i = 0; i < NB; ++i) {
            const float a0 = fast_exp2(sc[i][0] + b0), a1 = fast_exp2(sc[i][1] + b0);
            const float c0 = fast_exp2(sc[i][2] + b1), c1 = fast_exp2(sc[i][3] + b1);
            l0 += a0 + a1;
            l1 += c0 + c1;
            pf[i / 2][(i & 1) * 2] = pack2<kF16>(a0, a1);
            pf[i / 2][(i & 1) * 2 + 1] = pack2<kF16>(c0, c1);
        }
#pragma unroll
        for (int i = 0; i < NB / 2; ++i) {
#pragma unroll
            for (int n = 0; n < D / 16; ++n) {
                const int key = i * 16 + (((lane >> 3) & 1) << 3) + (lane & 7);
                const int ch = n * 2 + (lane >> 4);
                uint32_t r[4];
                ldsm4_t(vst + (uint32_t)key * C::kRow + (uint32_t)((ch ^ (key & 7)) << 4), r);
                mma16816<kF16>(acc[2 * n], pf[i], r[0], r[1]);
                mma16816<kF16>(acc[2 * n + 1], pf[i], r[2], r[3]);
            }
        }
        __syncwarp();  // the next load overwrites this stage
    }
    cp_async_wait<0>();
    __syncwarp();

    // ---- join of the warps, in the space of their stages
    l0 += __shfl_xor_sync(0xffffffffu, l0, 1);
    l1 += __shfl_xor_sync(0xffffffffu, l1, 1);
    l0 += __shfl_xor_sync(0xffffffffu, l0, 2);
    l1 += __shfl_xor_sync(0xffffffffu, l1, 2);
    constexpr int kPitch = D + 4;  // floats; the four extra spread the rows over the banks
    __shared__ float sm_m[W][16], sm_l[W][16];
    float* o = reinterpret_cast<float*>(mine);
#pragma unroll
    for (int i = 0; i < D / 8; ++i) {
        const int col = i * 8 + (lane & 3) * 2;
        *reinterpret_cast<float2*>(o + (lane >> 2) * kPitch + col) = make_float2(acc[i][0], acc[i][1]);
        *reinterpret_cast<float2*>(o + ((lane >> 2) + 8) * kPitch + col) = make_float2(acc[i][2], acc[i][3]);
    }
    if ((lane & 3) == 0) {
        sm_m[warp][lane >> 2] = m0;
        sm_m[warp][(lane >> 2) + 8] = m1;
        sm_l[warp][lane >> 2] = l0;
        sm_l[warp][(lane >> 2) + 8] = l1;
    }
    __syncthreads();
    const int rows = min(16, p.q_rows - rt * 16);
    for (int i = threadIdx.x; i < rows * (D / 4); i += W * 32) {
        const int r = i / (D / 4), col = i % (D / 4) * 4;
        float m = sm_m[0][r];
#pragma unroll
        for (int w = 1; w < W; ++w) m = fmaxf(m, sm_m[w][r]);
        float l = 0.f, y[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int w = 0; w < W; ++w) {
            // All keys masked: the sum is an exact zero (and not NaN, as of a row of NaN scores).
            if (sm_l[w][r] == 0.f) continue;
            const float f = fast_exp2(sm_m[w][r] - m);
            const float4 x = *reinterpret_cast<const float4*>(reinterpret_cast<const float*>(smem + w * C::kWarpBytes) +
                                                              r * kPitch + col);
            l += f * sm_l[w][r];
            y[0] += f * x.x;
            y[1] += f * x.y;
            y[2] += f * x.z;
            y[3] += f * x.w;
        }
        const bool empty = l == 0.f;
        const float inv = empty ? 0.f : 1.f / l;
        const float lse2 = empty ? -INFINITY : m - kShift + __log2f(l);
        const size_t row = row_base + rt * 16 + r;
        if (p.part_o) {
            const size_t at = (size_t)split * p.rows + row;
            // combine_kernel does not read the output of an empty part.
            if (!empty)
                *reinterpret_cast<float4*>(p.part_o + at * D + col) =
                    make_float4(y[0] * inv, y[1] * inv, y[2] * inv, y[3] * inv);
            if (col == 0) p.part_lse[at] = lse2;
        } else {
            *reinterpret_cast<uint2*>(reinterpret_cast<uint16_t*>(p.out) + row * D + col) =
                make_uint2(pack2<kF16>(y[0] * inv, y[1] * inv), pack2<kF16>(y[2] * inv, y[3] * inv));
            if (col == 0 && p.lse) p.lse[row] = lse2 * 0.69314718055994531f;
        }
    }
    if (p.beside && blockIdx.x == gridDim.x - 1 && blockIdx.y == gridDim.y - 1) griddep_wait();
}

struct CombineParams {
    const float* o[2];    // two sets of parts: [n][rows][D]
    const float* lse[2];  // [n][rows], log2
    int n[2];
    void* out;
    float* lse_out;
    long long rows;
};

// Up to 32 parts: one warp per row, lane i with part i's weight, no barrier.
template <int D, bool kF16>
__global__ void __launch_bounds__(128) combine_few_kernel(const CombineParams p) {
    griddep_wait();
    const long long row = (long long)blockIdx.x * 4 + (threadIdx.x >> 5);
    if (row >= p.rows) return;
    const int lane = threadIdx.x & 31;
    constexpr int E = D / 32;
    const int total = p.n[0] + p.n[1];
    float x = -INFINITY;
    if (lane < p.n[0])
        x = p.lse[0][(size_t)lane * p.rows + row];
    else if (lane < total)
        x = p.lse[1][(size_t)(lane - p.n[0]) * p.rows + row];
    float m = x;
#pragma unroll
    for (int s = 16; s > 0; s >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, s));
    const float mine = x == -INFINITY ? 0.f : fast_exp2(x - m);
    float y[E], l = 0.f;
#pragma unroll
    for (int e = 0; e < E; ++e) y[e] = 0.f;
    constexpr int kBatch = 8;  // loads in flight
    for (int i0 = 0; i0 < total; i0 += kBatch) {
        float a[kBatch][E];
#pragma unroll
        for (int k = 0; k < kBatch; ++k) {
            const int i = min(i0 + k, total - 1);
            const float* src = (i < p.n[0] ? p.o[0] + ((size_t)i * p.rows + row) * D
                                           : p.o[1] + ((size_t)(i - p.n[0]) * p.rows + row) * D) + lane * E;
            if constexpr (E == 4) {
                const float4 v = *reinterpret_cast<const float4*>(src);
                a[k][0] = v.x, a[k][1] = v.y, a[k][2] = v.z, a[k][3] = v.w;
            } else {
                const float2 v = *reinterpret_cast<const float2*>(src);
                a[k][0] = v.x, a[k][1] = v.y;
            }
        }
#pragma unroll
        for (int k = 0; k < kBatch; ++k) {
            const float w = i0 + k < total ? __shfl_sync(0xffffffffu, mine, (i0 + k) & 31) : 0.f;
            l += w;
            // Weight 0: no visible key (that output was not written), or nothing beside the largest.
#pragma unroll
            for (int e = 0; e < E; ++e) y[e] += w == 0.f ? 0.f : w * a[k][e];
        }
    }
    const bool any = l > 0.f || l != l;  // NaN stays NaN
    const float inv = any ? 1.f / l : 0.f;
    uint32_t* out = reinterpret_cast<uint32_t*>(p.out) + row * (D / 2) + lane * (E / 2);
#pragma unroll
    for (int e = 0; e < E / 2; ++e) out[e] = pack2<kF16>(y[2 * e] * inv, y[2 * e + 1] * inv);
    if (lane == 0 && p.lse_out) p.lse_out[row] = any ? (m + __log2f(l)) * 0.69314718055994531f : -INFINITY;
}

// One block per row, one warp per share of its parts: O = sum_i w_i O_i / sum_i w_i with
// w_i = 2^(lse_i - max). Parts without a visible key (-inf) weigh nothing, whatever their output holds.
constexpr int kJoinWarps = 8;
template <int D, bool kF16>
__global__ void __launch_bounds__(kJoinWarps * 32) combine_kernel(const CombineParams p) {
    griddep_wait();
    const long long row = blockIdx.x;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    constexpr int E = D / 32;
    __shared__ float sm_y[kJoinWarps][D], sm_l[kJoinWarps], sm_m[kJoinWarps];
    const int total = p.n[0] + p.n[1];
    auto lse_at = [&](int i) {
        return i < p.n[0] ? p.lse[0][(size_t)i * p.rows + row] : p.lse[1][(size_t)(i - p.n[0]) * p.rows + row];
    };
    float m = -INFINITY;
    for (int i = threadIdx.x; i < total; i += kJoinWarps * 32) m = fmaxf(m, lse_at(i));
#pragma unroll
    for (int s = 16; s > 0; s >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, s));
    if (lane == 0) sm_m[warp] = m;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < kJoinWarps; ++w) m = fmaxf(m, sm_m[w]);
    float y[E], l = 0.f;
#pragma unroll
    for (int e = 0; e < E; ++e) y[e] = 0.f;
    constexpr int kBatch = 4;  // loads in flight
    for (int i0 = warp; i0 < total; i0 += kJoinWarps * kBatch) {
        float a[kBatch][E], x[kBatch];
#pragma unroll
        for (int k = 0; k < kBatch; ++k) {
            const int j = i0 + k * kJoinWarps, i = min(j, total - 1);
            x[k] = j < total ? lse_at(i) : -INFINITY;
            const float* src = (i < p.n[0] ? p.o[0] + ((size_t)i * p.rows + row) * D
                                           : p.o[1] + ((size_t)(i - p.n[0]) * p.rows + row) * D) + lane * E;
            if constexpr (E == 4) {
                const float4 v = *reinterpret_cast<const float4*>(src);
                a[k][0] = v.x, a[k][1] = v.y, a[k][2] = v.z, a[k][3] = v.w;
            } else {
                const float2 v = *reinterpret_cast<const float2*>(src);
                a[k][0] = v.x, a[k][1] = v.y;
            }
        }
#pragma unroll
        for (int k = 0; k < kBatch; ++k) {
            const float w = x[k] == -INFINITY ? 0.f : fast_exp2(x[k] - m);
            l += w;
            // Weight 0: no visible key (that output was not written), or nothing beside the largest.
#pragma unroll
            for (int e = 0; e < E; ++e) y[e] += w == 0.f ? 0.f : w * a[k][e];
        }
    }
#pragma unroll
    for (int e = 0; e < E; ++e) sm_y[warp][lane * E + e] = y[e];
    if (lane == 0) sm_l[warp] = l;
    __syncthreads();
    if (threadIdx.x < D / 2) {
        const int c = threadIdx.x * 2;
        float sum = 0.f, a = 0.f, b = 0.f;
#pragma unroll
        for (int w = 0; w < kJoinWarps; ++w) {
            sum += sm_l[w];
            a += sm_y[w][c];
            b += sm_y[w][c + 1];
        }
        const bool any = sum > 0.f || sum != sum;  // NaN stays NaN
        const float inv = any ? 1.f / sum : 0.f;
        reinterpret_cast<uint32_t*>(p.out)[row * (D / 2) + threadIdx.x] = pack2<kF16>(a * inv, b * inv);
        if (threadIdx.x == 0 && p.lse_out) p.lse_out[row] = any ? (m + __log2f(sum)) * 0.69314718055994531f : -INFINITY;
    }
}

}  // namespace dec
}  // namespace bfk

namespace {

constexpr float kLog2e = 1.4426950408889634f;
// Up to so many bytes, counted anew for each sequence, a prefix is read with the sequences' own
// keys (from L2, after the first) by one kernel: us in a graph so / with the prefix's own kernel,
//   2.3 MB (B=4 Hq=8 Hkv=2 P=1000 d=64) 5.6 / 7.9     17 MB (B=1 Hq=8 Hkv=8 P=4096 d=128) 8.2 / 13.5
//   30 MB (B=16 Hq=32 Hkv=8 P=200 d=128) 10.5 / 10.3  41 MB (B=8 Hq=32 Hkv=8 P=1000 d=128) 12.2 / 10.8
// and one launch less, which is 3 us of the host's.
constexpr long long kTogetherBytes = 32LL << 20;

// How a step is split. A function of its sizes alone, so that the workspace can be sized
// ahead of the call.
struct Plan {
    long long rows;
    int row_tiles;        // 16-row tiles of a KV head
    int chunk, splits;    // cache: keys of a split, splits
    int p_splits, p_tiles;  // prefix: splits, KV tiles of a split
    bool together;        // the prefix's keys are read with each sequence's own, by one kernel
    bool wide;            // blocks of kWideWarps warps
    bool direct;          // one split, no prefix part: the kernel writes O itself
    long long bytes;
};

int make_plan(int B, int Hq, int Hkv, int T, int P, int C, int d, int window, int sinks, Plan* out) {
    if (B <= 0 || Hq <= 0 || Hkv <= 0 || T <= 0) return bf_set_error(BF_ERR_ARG, "empty problem: B, H and T must be >= 1");
    if (Hq % Hkv) return bf_set_error(BF_ERR_ARG, "query heads must be a multiple of KV heads");
    if (d != 64 && d != 128) return bf_set_error(BF_ERR_ARG, "BlackFlash supports d=64 and d=128");
    if (P < 0 || C < 0 || P > (1 << 30) || C > (1 << 30)) return bf_set_error(BF_ERR_ARG, "need 0 .. 2^30 keys");
    if (P == 0 && C == 0) return bf_set_error(BF_ERR_ARG, "no prefix and no cache");
    if (window < 1 || sinks < 0) return bf_set_error(BF_ERR_ARG, "need window >= 1 and sinks >= 0");
    Plan& p = *out;
    const long long q_rows = (long long)(Hq / Hkv) * T;
    // Checked by division: three factors of 31 bits pass 64, and `units` below is a divisor.
    if (q_rows > (1 << 20) || (long long)B * Hq > 0x7fffffffLL / T) return bf_set_error(BF_ERR_ARG, "too many query rows");
    p.rows = (long long)B * Hq * T;
    p.row_tiles = (int)((q_rows + 15) / 16);
    const long long units = (long long)B * Hkv * p.row_tiles;
    // The longest run of keys a row tile can see.
    long long vis = (long long)window + T - 1 + sinks;
    if (vis > C) vis = C;
    // A short prefix is not worth a kernel of its own, which reads it once for the batch but
    // takes a launch, its start and parts to join.
    p.together = P > 0 && P + vis <= kTogetherBytes / (d * 4) / units;
    if (p.together) vis += P;
    // Splits: blocks run three a multiprocessor, a unit's splits one grid row after the other, so
    // that the last, shorter ones fill up what the others leave. The time of a chunk size, in
    // keys of streaming: the work over the slots and a last block, at least one block; `start`
    // is what a block's start and join take. Candidates fill one to six waves, evenly or
    // with a short last split.
    const long long slots = 3 * kPlanSms, start = 16384 / d;
    long long best = -1;
    p.chunk = 128;
    p.splits = 0;
    for (int i = 0; i < 20 && vis > 0; ++i) {
        const int k = i / 2;
        const long long want = k < 4 ? k + 1 : (k - 3) * slots / units;
        if (want < 1) continue;
        long long chunk = (vis + want - 1) / want;
        if (i & 1) chunk += chunk / 4;
        chunk = (chunk + 127) / 128 * 128;
        const long long n = (vis + chunk - 1) / chunk, last = vis - (n - 1) * chunk;
        long long cost = n * units <= slots ? slots * ((n > 1 ? chunk : vis) + start)
                                            : units * (vis + n * start) + slots * (last + start);
        if (n > 1) cost += slots * start;  // the join's launch (256 keys at d = 64: 4.1 -> 3.4 us)
        if (best < 0 || cost < best) {
            best = cost;
            p.chunk = (int)chunk;
            p.splits = (int)n;
        }
    }
    // Few keys: one block of eight warps a unit and no join. That saves the parts' way through
    // memory and a launch, which is 3.1 us of the host's where calls follow one another and nothing
    // in a graph; but it leaves the other multiprocessors idle. us in a graph, split / wide, by
    // steps a warp (256 keys at d = 64, 128 at d = 128):
    //                        2           3           4           6            8
    //   d=64,   1 unit    4.5 / 4.3   4.3 / 5.3   4.5 / 6.5   5.3 / 8.5    5.5 / 10.7
    //          48 units   5.7 / 4.6   6.0 / 5.7   6.3 / 6.8   7.0 / 8.9    7.6 / 11.0
    //          96 units   6.4 / 4.7   6.9 / 5.9   7.6 / 7.0   8.9 / 9.1   10.4 / 11.3
    //         144 units   7.3 / 4.7   7.7 / 5.8   8.9 / 6.9  10.4 / 9.1   13.3 / 11.3
    //   d=128,  1 unit    4.9 / 4.6   5.3 / 5.6   5.5 / 6.7   5.7 / 8.7    5.5 / 10.8
    //          48 units   5.3 / 4.8   6.3 / 6.1   7.0 / 7.1   7.7 / 9.1    8.3 / 11.1
    //          96 units   6.7 / 5.0   7.6 / 6.1   8.4 / 7.2   9.6 / 9.3   11.2 / 11.4
    //         144 units   7.5 / 5.0  10.1 / 6.1   9.5 / 7.2  12.8 / 9.3   15.4 / 11.4
    // From 48 units on wide is taken for units / 16 steps, up to which it is no slower in a graph
    // either (3 % at most). Below that for three: the third step costs up to 1 us in a graph at d = 64
    // (0.3 at d = 128) and spares calls outside of one their second launch (9.1 -> 5.9 us); a fourth
    // would cost 2 us for the same.
    const long long keys = 2048 / d, steps = (vis + bfk::dec::kWideWarps * keys - 1) / (bfk::dec::kWideWarps * keys);
    p.wide = units <= kPlanSms && vis > bfk::dec::kWarps * keys && steps <= (units > 48 ? units / 16 : 3);
    if (p.wide) {
        p.splits = 1;
        p.chunk = (int)vis;
    }
    p.p_splits = p.p_tiles = 0;
    if (P > 0 && !p.together) {
        const long long per = 128 / q_rows;
        const long long tiles = per ? (B + per - 1) / per : B * ((q_rows + 127) / 128);
        const long long u = (tiles + 1) / 2 * Hkv;
        const int nk = (P + 127) / 128;
        // The prefix blocks keep a multiprocessor each, bound by their steps; the cache's part,
        // bound by bytes, runs on the others meanwhile and on all of them after. The split that
        // ends first, in ns as measured: a step of two 128-row tiles, a block's start and end,
        // the bytes a multiprocessor streams (the caches half full), a part's write and read.
        const long long step = d == 128 ? 2200 : 1300, ends = 5000;
        const double cache = floor((double)B * Hkv * C * d * 2 / 50);  // ns of one multiprocessor
        best = -1;
        for (int n = 1; n <= nk && n <= 2 * kPlanSms; n += 1 + n / 16) {
            const int s = (nk + n - 1) / n, real = (nk + s - 1) / s;
            const long long blocks = real * u, used = blocks < kPlanSms ? blocks : kPlanSms;
            const long long t = (blocks + kPlanSms - 1) / kPlanSms * (s * step + ends);
            const double meanwhile = (double)((kPlanSms - used) * t);
            const long long after = cache > meanwhile ? (long long)((cache - meanwhile) / kPlanSms) : 0;
            const long long cost = t + after + real * p.rows * d * 8 / 3000;
            if (best < 0 || cost < best) {
                best = cost;
                p.p_splits = real;
                p.p_tiles = s;
            }
        }
    }
    p.direct = p.p_splits == 0 && p.splits == 1;
    p.bytes = p.direct ? 0 : (long long)(p.splits + p.p_splits) * p.rows * (d + 1) * 4;
    return BF_OK;
}

template <int D, bool kF16, bool kPrefix, int W>
int launch_warps(const bfk::dec::Params& p, int splits, long long units, cudaStream_t stream) {
    static std::atomic<bool> done[64];  // per device; zero-initialised (static storage)
    int rc;
    auto kernel = bfk::dec::decode_kernel<D, kF16, kPrefix, W>;
    constexpr int smem = bfk::dec::Cfg<D, W>::kSmem;
    if ((rc = allow_smem(kernel, smem, done)) != BF_OK) return rc;
    return launch_error(launch_pdl(kernel, dim3((unsigned)units, (unsigned)splits), W * 32, smem, stream, p));
}

template <int D, bool kF16, bool kPrefix>
int launch_decode(const bfk::dec::Params& p, const Plan& plan, long long units, cudaStream_t stream) {
    return plan.wide ? launch_warps<D, kF16, kPrefix, bfk::dec::kWideWarps>(p, plan.splits, units, stream)
                     : launch_warps<D, kF16, kPrefix, bfk::dec::kWarps>(p, plan.splits, units, stream);
}

struct StepArgs {
    const void* q;
    const bf_view *kp, *vp, *k, *v;
    const int* lengths;
    void* o;
    float* lse;
    void* ws;
    long long ws_bytes;
    int B, Hq, Hkv, T, P, C, d, window, sinks, dtype;
    float scale;
    cudaStream_t stream;
};

int decode_step(const StepArgs& a) {
    Plan plan;
    int rc;
    if ((rc = make_plan(a.B, a.Hq, a.Hkv, a.T, a.P, a.C, a.d, a.window, a.sinks, &plan)) != BF_OK) return rc;
    if (a.dtype != BF_DTYPE_BF16 && a.dtype != BF_DTYPE_F16) return bf_set_error(BF_ERR_ARG, "dtype must be bf16 or fp16");
    if (!(a.scale > 0.f) || !isfinite(a.scale)) return bf_set_error(BF_ERR_ARG, "scale must be positive and finite");
    if (!a.q || !a.o || ((reinterpret_cast<uintptr_t>(a.q) | reinterpret_cast<uintptr_t>(a.o)) & 15u))
        return bf_set_error(BF_ERR_ARG, "Q and O must be non-null and 16-byte aligned");
    if (a.C > 0 && !a.lengths) return bf_set_error(BF_ERR_ARG, "lengths: null pointer");
    if (plan.bytes > 0 && (!a.ws || a.ws_bytes < plan.bytes || (reinterpret_cast<uintptr_t>(a.ws) & 31u)))
        return bf_set_error(BF_ERR_ARG, "workspace null, misaligned or smaller than blackflash_decode_workspace_bytes()");
    const bool f16 = a.dtype == BF_DTYPE_F16;
    float* part_o = reinterpret_cast<float*>(a.ws);
    const long long parts = plan.splits + plan.p_splits;
    float* part_lse = part_o + parts * plan.rows * a.d;
    ViewStrides sk, sv;
    if (a.C > 0) {
        if ((rc = check_view(a.k, "K_cache", a.B, a.Hkv, a.C, a.d, 2, &sk)) != BF_OK) return rc;
        if ((rc = check_view(a.v, "V_cache", a.B, a.Hkv, a.C, a.d, 2, &sv)) != BF_OK) return rc;
    }
    ViewStrides skp, svp;
    if (a.P > 0) {
        if ((rc = check_view(a.kp, "K_prefix", 1, a.Hkv, a.P, a.d, 2, &skp)) != BF_OK) return rc;
        if ((rc = check_view(a.vp, "V_prefix", 1, a.Hkv, a.P, a.d, 2, &svp)) != BF_OK) return rc;
    }
    if (a.P > 0 && !plan.together) {
        if ((rc = bind_context()) != BF_OK) return rc;
        PrefixArgs x;
        memset(&x, 0, sizeof(x));
        x.q = a.q;
        x.k = *a.kp;
        x.v = *a.vp;
        x.o = part_o + (long long)plan.splits * plan.rows * a.d;
        x.lse2 = part_lse + (long long)plan.splits * plan.rows;
        x.B = a.B;
        x.Hq = a.Hq;
        x.Hkv = a.Hkv;
        x.T = a.T;
        x.P = a.P;
        x.d = a.d;
        x.f16 = f16;
        x.scale = a.scale;
        x.splits = plan.p_splits;
        x.split_tiles = plan.p_tiles;
        x.stream = a.stream;
        if ((rc = bf_prefix_partial(x)) != BF_OK) return rc;
    }
    if (a.C > 0 || plan.together) {
        bfk::dec::Params p;
        memset(&p, 0, sizeof(p));
        p.q = a.q;
        if (a.C > 0) {
            p.k = reinterpret_cast<const char*>(a.k->data);
            p.v = reinterpret_cast<const char*>(a.v->data);
            for (int i = 0; i < 3; ++i) {
                p.ks[i] = sk.s[i] * 2;
                p.vs[i] = sv.s[i] * 2;
            }
        }
        if (plan.together) {
            p.kp = reinterpret_cast<const char*>(a.kp->data);
            p.vp = reinterpret_cast<const char*>(a.vp->data);
            for (int i = 0; i < 2; ++i) {
                p.kps[i] = skp.s[i + 1] * 2;
                p.vps[i] = svp.s[i + 1] * 2;
            }
            p.prefix = a.P;
        }
        p.lengths = a.lengths;
        p.out = a.o;
        p.lse = a.lse;
        p.part_o = plan.direct ? nullptr : part_o;
        p.part_lse = plan.direct ? nullptr : part_lse;
        p.rows = plan.rows;
        p.hkv = a.Hkv;
        p.q_rows = a.Hq / a.Hkv * a.T;
        p.tokens = a.T;
        p.cap = a.C;
        p.row_tiles = plan.row_tiles;
        p.window = a.window < a.C ? a.window : a.C;
        p.sinks = a.sinks < a.C ? a.sinks : a.C;
        p.chunk = plan.chunk;
        p.beside = a.P > 0 && !plan.together;
        p.scale_log2 = a.scale * kLog2e;
        const long long units = (long long)a.B * a.Hkv * plan.row_tiles;
        using Launch = int (*)(const bfk::dec::Params&, const Plan&, long long, cudaStream_t);
        const Launch launch[2][2][2] = {  // [d == 128][fp16][prefix among the keys]
            {{launch_decode<64, false, false>, launch_decode<64, false, true>},
             {launch_decode<64, true, false>, launch_decode<64, true, true>}},
            {{launch_decode<128, false, false>, launch_decode<128, false, true>},
             {launch_decode<128, true, false>, launch_decode<128, true, true>}}};
        rc = launch[a.d == 128][f16][plan.together](p, plan, units, a.stream);
        if (rc != BF_OK || plan.direct) return rc;
    }
    bfk::dec::CombineParams c;
    c.o[0] = part_o;
    c.lse[0] = part_lse;
    c.n[0] = plan.splits;
    c.o[1] = part_o + (long long)plan.splits * plan.rows * a.d;
    c.lse[1] = part_lse + (long long)plan.splits * plan.rows;
    c.n[1] = plan.p_splits;
    c.out = a.o;
    c.lse_out = a.lse;
    c.rows = plan.rows;
    // A block per row where there are more parts than lanes: 128 parts of 32 rows took 9 us by
    // one warp a row; 18 parts of 2048 rows take 10.5 us by a block a row, 4 by a warp.
    if (plan.splits + plan.p_splits <= 32) {
        auto kernel = a.d == 64 ? (f16 ? bfk::dec::combine_few_kernel<64, true> : bfk::dec::combine_few_kernel<64, false>)
                                : (f16 ? bfk::dec::combine_few_kernel<128, true> : bfk::dec::combine_few_kernel<128, false>);
        return launch_error(launch_pdl(kernel, dim3((unsigned)((plan.rows + 3) / 4)), 128, 0, a.stream, c));
    }
    auto kernel = a.d == 64 ? (f16 ? bfk::dec::combine_kernel<64, true> : bfk::dec::combine_kernel<64, false>)
                            : (f16 ? bfk::dec::combine_kernel<128, true> : bfk::dec::combine_kernel<128, false>);
    return launch_error(launch_pdl(kernel, dim3((unsigned)plan.rows), bfk::dec::kJoinWarps * 32, 0, a.stream, c));
}

}  // namespace

extern "C" long long blackflash_decode_workspace_bytes(int B, int Hq, int Hkv, int T, int P, int C, int d, int window,
                                                       int sinks) {
    bf_set_error(BF_OK, "");
    Plan plan;
    return make_plan(B, Hq, Hkv, T, P, C, d, window, sinks, &plan) == BF_OK ? plan.bytes : -1;
}

extern "C" int blackflash_window_decode(const void* Q, const bf_view* K, const bf_view* V, const int* lengths, void* O,
                                        float* lse, void* workspace, long long workspace_bytes, int B, int Hq, int Hkv,
                                        int T, int C, int d, int window, int sinks, float scale, int dtype, void* stream) {
    bf_set_error(BF_OK, "");
    const StepArgs a = {Q, nullptr, nullptr, K, V, lengths, O, lse, workspace, workspace_bytes, B, Hq, Hkv, T, 0, C, d,
                        window, sinks, dtype, scale, reinterpret_cast<cudaStream_t>(stream)};
    return decode_step(a);
}

extern "C" int blackflash_prefix_decode(const void* Q, const bf_view* Kp, const bf_view* Vp, const bf_view* K,
                                        const bf_view* V, const int* lengths, void* O, float* lse, void* workspace,
                                        long long workspace_bytes, int B, int Hq, int Hkv, int T, int P, int C, int d,
                                        float scale, int dtype, void* stream) {
    bf_set_error(BF_OK, "");
    const StepArgs a = {Q, Kp, Vp, K, V, lengths, O, lse, workspace, workspace_bytes, B, Hq, Hkv, T, P, C, d,
                        0x7fffffff, 0, dtype, scale, reinterpret_cast<cudaStream_t>(stream)};
    return decode_step(a);
}
