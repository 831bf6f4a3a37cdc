// Checks and tensor maps of the strided [batch, heads, tokens, d] views that the
// position-aware operators take (bf_view in include/blackflash_b200.h).
#pragma once
#include "launch_sm100.h"

// B200 only: the split plans use this count, so that a workspace's size does not depend on
// the device that happens to be current.
constexpr int kPlanSms = 148;

// Strides of a view with those of one-element axes (which mean nothing) replaced.
struct ViewStrides {
    long long s[3];
};

// 16-byte rows and starts, no broadcast (zero) or negative strides.
inline int check_view(const bf_view* v, const char* name, long long n0, long long n1, long long n2, int d,
                      int elem_bytes, ViewStrides* out) {
    char msg[160];
    if (!v || !v->data) {
        snprintf(msg, sizeof(msg), "%s: null pointer", name);
        return bf_set_error(BF_ERR_ARG, msg);
    }
    if (reinterpret_cast<uintptr_t>(v->data) & 15u) {
        snprintf(msg, sizeof(msg), "%s must be 16-byte aligned", name);
        return bf_set_error(BF_ERR_ARG, msg);
    }
    const long long n[3] = {n0, n1, n2};
    for (int i = 0; i < 3; ++i) {
        out->s[i] = n[i] > 1 ? v->stride[i] : d;
        if (out->s[i] <= 0 || out->s[i] * elem_bytes % 16 || out->s[i] >= (1LL << 36)) {
            snprintf(msg, sizeof(msg), "%s: strides must be positive multiples of 16 bytes (axis %d has %lld elements)", name,
                     i, v->stride[i]);
            return bf_set_error(BF_ERR_ARG, msg);
        }
    }
    return BF_OK;
}

// Makes the current device's primary context current to the calling thread: the tensor-map
// encode is a driver call, and a thread that has only used the runtime implicitly (torch's
// autograd worker) may not have one yet.
inline int bind_context() {
    int cur = 0;
    if (cudaGetDevice(&cur) != cudaSuccess || cudaSetDevice(cur) != cudaSuccess)
        return bf_set_error(BF_ERR_CUDA, "no CUDA device context");
    return BF_OK;
}

// 4-D map {d, tokens, heads, batch} of 16-bit elements with 128-byte swizzle and boxes of
// 64 columns x box1 x box2. Coordinates past an axis read as zero.
inline int make_map_4d(CUtensorMap* m, const void* base, bool f16, const long long dim[4], const long long stride[3],
                       int box1, int box2) {
    PFN_encodeTiled enc = get_encode_fn();
    if (!enc) return bf_set_error(BF_ERR_CUDA, "cuTensorMapEncodeTiled is unavailable");
    cuuint64_t dims[4] = {(cuuint64_t)dim[0], (cuuint64_t)dim[1], (cuuint64_t)dim[2], (cuuint64_t)dim[3]};
    cuuint64_t strides[3] = {(cuuint64_t)stride[0] * 2, (cuuint64_t)stride[1] * 2, (cuuint64_t)stride[2] * 2};
    cuuint32_t box[4] = {64, (cuuint32_t)box1, (cuuint32_t)box2, 1};
    cuuint32_t estr[4] = {1, 1, 1, 1};
    const CUresult r = enc(m, f16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 4,
                           const_cast<void*>(base), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
                           CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (r != CUDA_SUCCESS) {
        char msg[200];
        snprintf(msg, sizeof(msg), "cuTensorMapEncodeTiled rejected the tensor (error %d, base %p, tokens %lld, heads %lld)",
                 (int)r, base, dim[1], dim[2]);
        return bf_set_error(BF_ERR_CUDA, msg);
    }
    return BF_OK;
}

// Raises a kernel's dynamic shared memory limit once per device.
template <typename K>
int allow_smem(K kernel, int bytes, std::atomic<bool> (&done)[64]) {
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return bf_set_error(BF_ERR_CUDA, "cudaGetDevice failed");
    if (!done[dev]) {
        const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
        if (e != cudaSuccess) return bf_set_error(BF_ERR_CUDA, cudaGetErrorString(e));
        done[dev] = true;
    }
    return BF_OK;
}

inline int launch_error(cudaError_t e) {
    if (e == cudaSuccess) e = cudaGetLastError();
    return e == cudaSuccess ? BF_OK : bf_set_error(BF_ERR_CUDA, cudaGetErrorString(e));
}

// The prefix part of a decoding step: every query row of Q (contiguous [B, Hq, T, d])
// against the KV tiles of Kp, Vp [Hkv, P, d], `splits` ranges of `split_tiles` tiles each.
// Writes fp32 O [splits][B * Hq * T][d], normalised over its range, and log2-sum-exp2.
struct PrefixArgs {
    const void* q;
    bf_view k, v;  // axis 0 unused
    float* o;
    float* lse2;
    int B, Hq, Hkv, T, P, d, f16;
    float scale;
    int splits, split_tiles;
    cudaStream_t stream;
};
int bf_prefix_partial(const PrefixArgs& a);  // window_sm100.cu
