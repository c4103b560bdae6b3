// Parts of rows whose keys several blocks share, and the kernel that joins them.
#pragma once

#include "kv8.cuh"

// Part s of head h (its token counted from the call's first) is at index h * splits + s: `o` the output not yet
// divided, `ml` the maximum in powers of two and the sum; a part that saw no key has the maximum -inf.
struct Kv8Parts {
    float *o, *ml;
    int splits;
    // portions: the first of the entries' token bounds; null: the call's tokens are 0 .. count - 1
    const int* indptr;
    int count;
};
__device__ __forceinline__ int kv8_first_token(const Kv8Parts& p) { return p.indptr != nullptr ? p.indptr[0] : 0; }

// A warp a head.  Only the call's own tokens are touched.
template <typename A>
__global__ void __launch_bounds__(128) kv8_merge_kernel(Kv8Parts p, A* out, int nq, int hd) {
    pdl_launch_dependents();
    pdl_wait();
    const int first = kv8_first_token(p), end = p.indptr != nullptr ? p.indptr[p.count] : p.count;
    const int head = blockIdx.x * 4 + (threadIdx.x >> 5), lane = threadIdx.x & 31;
    if (head >= (end - first) * nq) return;
    const float* ml = p.ml + (size_t)head * p.splits * 2;
    float m = -INFINITY;
    for (int s = lane; s < p.splits; s += 32) m = fmaxf(m, ml[2 * s]);
    m = warp_max(m);
    const float ref = m == -INFINITY ? 0.f : m;
    float l = 0.f;
    for (int s = lane; s < p.splits; s += 32) l += ml[2 * s + 1] * exp2f(ml[2 * s] - ref);
    l = warp_sum(l);
    const float inv = l == 0.f ? 0.f : 1.f / l;
    for (int d = lane * 4; d < hd; d += 128) {
        float v[4] = {0.f, 0.f, 0.f, 0.f};
        for (int s = 0; s < p.splits; ++s) {
            const float w = exp2f(ml[2 * s] - ref);
            if (w == 0.f) continue;                        // a part without keys, or too small to matter
            float o[4];
            load4(p.o + ((size_t)head * p.splits + s) * hd + d, o);
#pragma unroll
            for (int i = 0; i < 4; ++i) v[i] = fmaf(w, o[i], v[i]);
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) v[i] *= inv;
        store4(out + ((size_t)first * nq + head) * hd + d, v);
    }
}

// `tokens`: at least as many as the call covers.
static inline int kv8_merge(const Kv8Parts& p, void* out, int act_dtype, int tokens, int nq, int hd, cudaStream_t s) {
    const dim3 grid((unsigned)(((long long)tokens * nq + 3) / 4));
    cudaError_t e;
    if (act_dtype == MSTAR_F32) e = mstar_launch((kv8_merge_kernel<float>), grid, dim3(128), 0, s, p, (float*)out, nq, hd);
    else e = mstar_launch((kv8_merge_kernel<bf16>), grid, dim3(128), 0, s, p, (bf16*)out, nq, hd);
    return e != cudaSuccess ? (int)e : launch_status();
}
