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
    // the tokens that there is room for; a portion longer than the caller said is left out beyond them
    int tokens;
};
__device__ __forceinline__ int kv8_first_token(const Kv8Parts& p) { return p.indptr != nullptr ? p.indptr[0] : 0; }
__device__ __forceinline__ bool kv8_has_room(const Kv8Parts& p, int token) { return token - kv8_first_token(p) < p.tokens; }

// A warp a head, eight parts' loads at a time (one after another, 64 parts of one token's 32 heads took 20 us).  Only
// the call's own tokens are touched.
template <typename A>
__global__ void __launch_bounds__(128) kv8_merge_kernel(Kv8Parts p, A* out, int nq, int hd) {
    pdl_launch_dependents();
    pdl_wait();
    const int first = kv8_first_token(p), end = p.indptr != nullptr ? p.indptr[p.count] : p.count;
    const int head = blockIdx.x * 4 + (threadIdx.x >> 5), lane = threadIdx.x & 31;
    if (head >= min(end - first, p.tokens) * nq) return;
    const float* ml = p.ml + (size_t)head * p.splits * 2;
    float m = -INFINITY;
    for (int s = lane; s < p.splits; s += 32) m = fmaxf(m, ml[2 * s]);
    m = warp_max(m);
    const float ref = m == -INFINITY ? 0.f : m;
    float l = 0.f;
    for (int s = lane; s < p.splits; s += 32) l += ml[2 * s + 1] * exp2f(ml[2 * s] - ref);
    l = warp_sum(l);
    const float inv = l == 0.f ? 0.f : 1.f / l;
    for (int d0 = 0; d0 < hd; d0 += 128) {
        const int d = min(d0 + lane * 4, hd - 4);
        const float* o = p.o + (size_t)head * p.splits * hd + d;
        float v[4] = {0.f, 0.f, 0.f, 0.f};
        for (int s0 = 0; s0 < p.splits; s0 += 8) {
            float part[8][4];
#pragma unroll
            for (int i = 0; i < 8; ++i) load4(o + (size_t)min(s0 + i, p.splits - 1) * hd, part[i]);
            const float w = (lane & 7) + s0 < p.splits ? exp2f(ml[2 * (s0 + (lane & 7))] - ref) : 0.f;
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const float wi = __shfl_sync(0xffffffffu, w, i);
                // a weight of zero is a part without keys, or one too small to matter; what lies there may be anything
#pragma unroll
                for (int j = 0; j < 4; ++j) v[j] = wi == 0.f ? v[j] : fmaf(wi, part[i][j], v[j]);
            }
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) v[i] *= inv;
        if (d0 + lane * 4 < hd) store4(out + ((size_t)first * nq + head) * hd + d, v);
    }
}

static inline int kv8_merge(const Kv8Parts& p, void* out, int act_dtype, int nq, int hd, cudaStream_t s) {
    const dim3 grid((unsigned)(((long long)p.tokens * nq + 3) / 4));
    cudaError_t e;
    if (act_dtype == MSTAR_F32) e = mstar_launch((kv8_merge_kernel<float>), grid, dim3(128), 0, s, p, (float*)out, nq, hd);
    else e = mstar_launch((kv8_merge_kernel<bf16>), grid, dim3(128), 0, s, p, (bf16*)out, nq, hd);
    return e != cudaSuccess ? (int)e : launch_status();
}
