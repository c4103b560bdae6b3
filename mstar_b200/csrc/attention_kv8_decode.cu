// Attention of single tokens over the 8-bit cache (format: kv8.cuh), bfloat16, head_dim 64, 128 or 256, any group of
// query heads and any page size.
//
// The work is the cache's bytes: a token reads each of its keys and values once for up to 8 query heads, some 4 flops
// a byte and head.  So the kernel is built around having loads in flight: every warp takes steps of 32 keys (16 at
// head_dim 256) straight from global memory into registers, keys of the step after next to the values being used, and
// nothing passes through shared memory on the way.  The products run on the tensor cores with the keys as rows, since
// 16 rows of queries would be mostly padding:
//   S^T [16 keys x 8 heads] += K [16 x 16] Q^T [16 x 8],   O^T [16 features x 8 heads] += V^T [16 x 16 keys] P^T.
// Which feature a fragment's element stands for is free as long as both operands agree, so that a thread's operands
// are runs of 16 bytes of a row: of K the features [16 t, 16 t + 16) and every 64 after them, of V [D/8 g, D/8 (g + 1))
// (lane = 4 g + t).  V's pairs of keys are put together by byte permutes, P^T comes from S^T by a matrix transpose
// between registers (movmatrix).
//
// e4m3 is exact in float16, so both products take float16: the queries are scaled by a power of two a head (their
// largest number into [1, 2); what falls below float16's range is 2^-25 of that), the weights lie in [0, 1].  The
// rows' scales are put on the scores: a key's by a product, and a value's as an addend of the exponent, since 2^s_j *
// 2^e_j v_j = 2^(s_j + e_j) v_j.  The weights of the values' product are therefore 2^(s_j + e_j - m') with a maximum m'
// of their own, so that they use float16's range whatever the values' scales are; the normaliser's are 2^(s_j - m).
//
// The steps of a (token, kv head) are dealt out in turn to the warps of a cluster of blocks, so that the lengths that
// are there decide the balance, not the bounds a launch was sized for.  The warps of a block are joined in shared
// memory, the blocks through distributed shared memory: one launch, no scratch memory, sums in a fixed order.
//
// Semantics are those of attention_generic.cu.
#include <cooperative_groups.h>
#include <cuda_fp16.h>

#include "kv8.cuh"

namespace cg = cooperative_groups;

struct Kv8DecodeArgs {
    const bf16* q;
    bf16* out;
    const uint8_t *codes, *scales;
    const int *block_table, *token_req, *cache_pos;
    int q_stride, bt_stride, pages, nq, nkv, window, keep_first, head_groups;
    float scale_log2e;
    PageSplit page;
};

__device__ __forceinline__ uint32_t e4m3x2_to_f16x2(uint32_t two) {
    uint32_t r;
    asm("{\n\t.reg .b16 lo, hi;\n\tmov.b32 {lo, hi}, %1;\n\tcvt.rn.f16x2.e4m3x2 %0, lo;\n\t}" : "=r"(r) : "r"(two));
    return r;
}
__device__ __forceinline__ uint32_t e4m3x2_hi_to_f16x2(uint32_t two) {
    uint32_t r;
    asm("{\n\t.reg .b16 lo, hi;\n\tmov.b32 {lo, hi}, %1;\n\tcvt.rn.f16x2.e4m3x2 %0, hi;\n\t}" : "=r"(r) : "r"(two));
    return r;
}
__device__ __forceinline__ void mma_f16_16816(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,
                                              uint32_t b0, uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};\n"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t transpose_8x8(uint32_t x) {
    uint32_t r;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(x));
    return r;
}
__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ uint32_t pack_f16(float lo, float hi) {
    const __half2 v = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&v);
}
// 2^(a - b) for maxima that may still be -inf (of a part without keys: 0)
__device__ __forceinline__ float ratio(float a, float b) { return a == -INFINITY ? 0.f : ex2(a - b); }

// what a thread holds of a step's rows
template <int D> struct ValueRun { uint4 w[D / 128]; };
template <> struct ValueRun<64> { uint2 w[1]; };

template <int D> __host__ __device__ constexpr int dec8_keys() { return D <= 128 ? 32 : 16; }          // keys of a step
template <int D> __host__ __device__ constexpr int dec8_most_warps() { return D <= 128 ? 12 : 8; }

template <int D>
__global__ void __launch_bounds__(32 * dec8_most_warps<D>(), 1) kv8_decode_kernel(Kv8DecodeArgs a) {
    constexpr int KEYS = dec8_keys<D>(), SUB = KEYS / 16;
    constexpr int KC = D / 64;             // 16-byte runs of a key row a thread holds
    constexpr int VW = D / 32;             // 4-byte words of a value row a thread holds
    constexpr int MT = D / 16;             // blocks of 16 features
    extern __shared__ __align__(16) float smem[];
    pdl_wait();
    cg::cluster_group cluster = cg::this_cluster();
    const int W = blockDim.x >> 5, warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    const int C = cluster.num_blocks(), rank = cluster.block_rank();
    const int pair = blockIdx.x / C, token = blockIdx.y;
    const int kvh = pair / a.head_groups, h0 = (pair % a.head_groups) * 8, G = a.nq / a.nkv, heads = min(8, G - h0);
    const int pos = a.cache_pos[token];
    const int* bt = a.block_table + (size_t)a.token_req[token] * a.bt_stride;
    const SeenKeys seen = seen_keys(pos, pos, a.window, a.keep_first);
    const uint32_t plane = (uint32_t)a.nkv * a.page.size;
    const uint8_t* codes = a.codes;

    // queries: head g, the features this thread's part of K has
    uint32_t qf[4 * KC][2];
    float head_scale;
    {
        const bool there = g < heads;
        const bf16* q = a.q + (size_t)token * a.q_stride + (size_t)(kvh * G + h0 + (there ? g : 0)) * D;
        float most = 0.f;
        uint32_t raw[KC][8];
#pragma unroll
        for (int c = 0; c < KC; ++c)
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                const uint4 w = *reinterpret_cast<const uint4*>(q + c * 64 + t * 16 + i * 8);
                raw[c][4 * i] = w.x; raw[c][4 * i + 1] = w.y; raw[c][4 * i + 2] = w.z; raw[c][4 * i + 3] = w.w;
            }
#pragma unroll
        for (int c = 0; c < KC; ++c)
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                if (!there) raw[c][i] = 0u;
                const float2 f = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&raw[c][i]));
                most = fmaxf(most, fmaxf(fabsf(f.x), fabsf(f.y)));
            }
        most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, 1));
        most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, 2));
        // the largest number's exponent, nothing where it has none (0, subnormal, not finite) or no inverse
        const uint32_t e = __float_as_uint(most) >> 23;
        const bool plain = e == 0 || e >= 254;
        const float down = plain ? 1.f : __uint_as_float((254u - e) << 23);
        head_scale = (plain ? 1.f : __uint_as_float(e << 23)) * a.scale_log2e;
#pragma unroll
        for (int c = 0; c < KC; ++c)
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
                for (int j = 0; j < 2; ++j) {
                    const float2 f = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&raw[c][2 * i + j]));
                    qf[c * 4 + i][j] = pack_f16(f.x * down, f.y * down);
                }
    }
    // of the two heads whose scores this thread has
    const float hs0 = __shfl_sync(0xffffffffu, head_scale, 8 * t), hs1 = __shfl_sync(0xffffffffu, head_scale, 8 * t + 4);

    float o[MT][4];
#pragma unroll
    for (int i = 0; i < MT; ++i) o[i][0] = o[i][1] = o[i][2] = o[i][3] = 0.f;
    float m0 = -INFINITY, m1 = -INFINITY, w0 = -INFINITY, w1 = -INFINITY, l0 = 0.f, l1 = 0.f;

    const int steps = (seen.count + KEYS - 1) / KEYS, stride = C * W;
    // the row (of the cache as a matrix of D bytes a row) of this lane's key of a step; keys past the last one are the
    // last one, and are masked
    auto row_of = [&](int step) -> uint32_t {
        const int v = min(step * KEYS + (lane & (KEYS - 1)), seen.count - 1);
        const int key = key_of(seen, v), logical = page_of(a.page, key);
        return ((uint32_t)page_id(bt, logical, a.bt_stride, a.pages) * 2 * a.nkv + kvh) * a.page.size +
               (uint32_t)(key - logical * a.page.size);
    };
    uint4 kr[2 * SUB][KC];                       // keys g, g + 8 of every 16
    ValueRun<D> vr[4 * SUB];                     // keys 2t, 2t + 1, 2t + 8, 2t + 9 of every 16
    auto load_keys = [&](uint32_t rows) {
#pragma unroll
        for (int i = 0; i < 2 * SUB; ++i) {
            const uint8_t* p = codes + (size_t)__shfl_sync(0xffffffffu, rows, g + 8 * i) * D + t * 16;
#pragma unroll
            for (int c = 0; c < KC; ++c) kr[i][c] = *reinterpret_cast<const uint4*>(p + c * 64);
        }
    };
    auto load_values = [&](uint32_t rows) {
#pragma unroll
        for (int i = 0; i < 4 * SUB; ++i) {
            const int key = (i >> 2) * 16 + 2 * t + (i & 1) + ((i & 2) << 2);
            const uint8_t* p = codes + (size_t)(__shfl_sync(0xffffffffu, rows, key) + plane) * D + g * (D / 8);
            vr[i] = *reinterpret_cast<const ValueRun<D>*>(p);
        }
    };
    auto load_scales = [&](uint32_t rows) -> uint32_t {
        return (uint32_t)a.scales[rows] | ((uint32_t)a.scales[(size_t)rows + plane] << 8);
    };

    int step = rank * W + warp;
    if (step < steps) {
        uint32_t rows = row_of(step), sc = load_scales(rows);
        load_keys(rows);
        load_values(rows);
        uint32_t next = step + stride < steps ? row_of(step + stride) : rows;
        for (; step < steps; step += stride) {
            const bool more = step + stride < steps;
            // ---- scores
            float s[SUB][4];
#pragma unroll
            for (int u = 0; u < SUB; ++u) {
                s[u][0] = s[u][1] = s[u][2] = s[u][3] = 0.f;
#pragma unroll
                for (int c = 0; c < KC; ++c) {
                    const uint32_t lo[4] = {kr[2 * u][c].x, kr[2 * u][c].y, kr[2 * u][c].z, kr[2 * u][c].w};
                    const uint32_t hi[4] = {kr[2 * u + 1][c].x, kr[2 * u + 1][c].y, kr[2 * u + 1][c].z, kr[2 * u + 1][c].w};
#pragma unroll
                    for (int i = 0; i < 4; ++i)
                        mma_f16_16816(s[u], e4m3x2_to_f16x2(lo[i]), e4m3x2_to_f16x2(hi[i]), e4m3x2_hi_to_f16x2(lo[i]),
                                      e4m3x2_hi_to_f16x2(hi[i]), qf[c * 4 + i][0], qf[c * 4 + i][1]);
                }
            }
            if (more) load_keys(next);
            // ---- weights; this thread has keys g, g + 8 of every 16 and heads 2t, 2t + 1
            float p[SUB][4];                     // exponents of the values' weights, then the weights
            float x0 = -INFINITY, x1 = -INFINITY, y0 = -INFINITY, y1 = -INFINITY;
#pragma unroll
            for (int u = 0; u < SUB; ++u)
#pragma unroll
                for (int k = 0; k < 2; ++k) {
                    const uint32_t two = __shfl_sync(0xffffffffu, sc, 16 * u + 8 * k + g);
                    const int ks = two & 255, vs = two >> 8;
                    const bool bad = ks == KV8_BAD_BYTE || vs == KV8_BAD_BYTE;
                    const float f = bad ? __int_as_float(0x7fc00000) : kv8_scale(ks);
                    const float e = (float)(vs - 127);
                    const bool in = step * KEYS + 16 * u + 8 * k + g < seen.count;
                    const float a0 = in ? s[u][2 * k] * f * hs0 : -INFINITY, a1 = in ? s[u][2 * k + 1] * f * hs1 : -INFINITY;
                    s[u][2 * k] = a0;
                    s[u][2 * k + 1] = a1;
                    p[u][2 * k] = a0 + e;
                    p[u][2 * k + 1] = a1 + e;
                    x0 = fmaxf(x0, a0);
                    x1 = fmaxf(x1, a1);
                    y0 = fmaxf(y0, a0 + e);
                    y1 = fmaxf(y1, a1 + e);
                }
#pragma unroll
            for (int d = 4; d < 32; d <<= 1) {
                x0 = fmaxf(x0, __shfl_xor_sync(0xffffffffu, x0, d));
                x1 = fmaxf(x1, __shfl_xor_sync(0xffffffffu, x1, d));
                y0 = fmaxf(y0, __shfl_xor_sync(0xffffffffu, y0, d));
                y1 = fmaxf(y1, __shfl_xor_sync(0xffffffffu, y1, d));
            }
            // (a maximum is -inf only where every score so far is NaN or -inf: the sums are NaN or zero then)
            x0 = fmaxf(m0, x0);
            x1 = fmaxf(m1, x1);
            y0 = fmaxf(w0, y0);
            y1 = fmaxf(w1, y1);
            l0 *= ratio(m0, x0);
            l1 *= ratio(m1, x1);
            const float r0 = ratio(w0, y0), r1 = ratio(w1, y1);
            if (__any_sync(0xffffffffu, (y0 != w0) | (y1 != w1))) {
#pragma unroll
                for (int i = 0; i < MT; ++i) {
                    o[i][0] *= r0;
                    o[i][1] *= r1;
                    o[i][2] *= r0;
                    o[i][3] *= r1;
                }
            }
            m0 = x0;
            m1 = x1;
            w0 = y0;
            w1 = y1;
            const float z0 = x0 == -INFINITY ? 0.f : x0, z1 = x1 == -INFINITY ? 0.f : x1;
            const float q0 = y0 == -INFINITY ? 0.f : y0, q1 = y1 == -INFINITY ? 0.f : y1;
            uint32_t pf[SUB][2];
#pragma unroll
            for (int u = 0; u < SUB; ++u)
#pragma unroll
                for (int k = 0; k < 2; ++k) {
                    l0 += ex2(s[u][2 * k] - z0);
                    l1 += ex2(s[u][2 * k + 1] - z1);
                    pf[u][k] = transpose_8x8(pack_f16(ex2(p[u][2 * k] - q0), ex2(p[u][2 * k + 1] - q1)));
                }
            // ---- values
#pragma unroll
            for (int u = 0; u < SUB; ++u) {
                const uint32_t* v0 = reinterpret_cast<const uint32_t*>(&vr[4 * u]);
                const uint32_t* v1 = reinterpret_cast<const uint32_t*>(&vr[4 * u + 1]);
                const uint32_t* v2 = reinterpret_cast<const uint32_t*>(&vr[4 * u + 2]);
                const uint32_t* v3 = reinterpret_cast<const uint32_t*>(&vr[4 * u + 3]);
#pragma unroll
                for (int j = 0; j < VW; ++j) {
                    // features 4j, 4j + 1 and 4j + 2, 4j + 3 of this thread's run, two keys side by side
                    const uint32_t a01 = __byte_perm(v0[j], v1[j], 0x5140), a23 = __byte_perm(v0[j], v1[j], 0x7362);
                    const uint32_t b01 = __byte_perm(v2[j], v3[j], 0x5140), b23 = __byte_perm(v2[j], v3[j], 0x7362);
                    mma_f16_16816(o[2 * j], e4m3x2_to_f16x2(a01), e4m3x2_hi_to_f16x2(a01), e4m3x2_to_f16x2(b01),
                                  e4m3x2_hi_to_f16x2(b01), pf[u][0], pf[u][1]);
                    mma_f16_16816(o[2 * j + 1], e4m3x2_to_f16x2(a23), e4m3x2_hi_to_f16x2(a23), e4m3x2_to_f16x2(b23),
                                  e4m3x2_hi_to_f16x2(b23), pf[u][0], pf[u][1]);
                }
            }
            if (more) {
                load_values(next);
                sc = load_scales(next);
                if (step + 2 * stride < steps) next = row_of(step + 2 * stride);
            }
        }
    }
    pdl_launch_dependents();

    // ---- the warps of the block: statistics (m, m', l) and outputs of 8 heads each
    constexpr int LD = D + 4;
#pragma unroll
    for (int d = 4; d < 32; d <<= 1) {
        l0 += __shfl_xor_sync(0xffffffffu, l0, d);
        l1 += __shfl_xor_sync(0xffffffffu, l1, d);
    }
    float* mine = smem;                                   // the block's own: [8][4]
    float* st_s = smem + 32;                              // [W][8][4]
    float* o_s = st_s + W * 32;                           // [W][8][LD], the block's own in the first warp's place
    if (g == 0) {
        float* st = st_s + warp * 32 + 2 * t * 4;
        st[0] = m0; st[1] = w0; st[2] = l0;
        st[4] = m1; st[5] = w1; st[6] = l1;
    }
    {
        float* dst = o_s + (size_t)warp * 8 * LD;
#pragma unroll
        for (int i = 0; i < MT; ++i) {
            const int d = g * (D / 8) + 2 * i;            // rows g and g + 8 of the block: two neighbouring features
            *reinterpret_cast<float2*>(dst + (2 * t) * LD + d) = make_float2(o[i][0], o[i][2]);
            *reinterpret_cast<float2*>(dst + (2 * t + 1) * LD + d) = make_float2(o[i][1], o[i][3]);
        }
    }
    __syncthreads();
    if (threadIdx.x < 8) {
        float m = -INFINITY, w = -INFINITY, l = 0.f;
        for (int i = 0; i < W; ++i) {
            m = fmaxf(m, st_s[i * 32 + threadIdx.x * 4]);
            w = fmaxf(w, st_s[i * 32 + threadIdx.x * 4 + 1]);
        }
        for (int i = 0; i < W; ++i) {
            float* st = st_s + i * 32 + threadIdx.x * 4;
            // (a warp whose every score was NaN has the maximum -inf and a sum of NaN)
            l += st[2] == 0.f ? 0.f : st[0] == -INFINITY ? st[2] : st[2] * ex2(st[0] - m);
            st[3] = ratio(st[1], w);
        }
        mine[threadIdx.x * 4] = m;
        mine[threadIdx.x * 4 + 1] = w;
        mine[threadIdx.x * 4 + 2] = l;
    }
    __syncthreads();
    for (int i = threadIdx.x; i < heads * (D / 4); i += blockDim.x) {
        const int h = i / (D / 4), d = (i % (D / 4)) * 4;
        float4 sum = make_float4(0.f, 0.f, 0.f, 0.f);
        for (int w = 0; w < W; ++w) {
            const float f = st_s[w * 32 + h * 4 + 3];
            const float4 x = *reinterpret_cast<const float4*>(o_s + (size_t)(w * 8 + h) * LD + d);
            sum.x = fmaf(x.x, f, sum.x);
            sum.y = fmaf(x.y, f, sum.y);
            sum.z = fmaf(x.z, f, sum.z);
            sum.w = fmaf(x.w, f, sum.w);
        }
        *reinterpret_cast<float4*>(o_s + (size_t)h * LD + d) = sum;       // (its own element of warp 0's part)
    }
    cluster.sync();
    // ---- the blocks of the cluster: each joins a share of the elements
    const int total = heads * (D / 4);
    for (int i = rank * blockDim.x + threadIdx.x; i < total; i += C * blockDim.x) {
        const int h = i / (D / 4), d = (i % (D / 4)) * 4;
        float m = -INFINITY, w = -INFINITY, l = 0.f;
        for (int c = 0; c < C; ++c) {
            const float* st = cluster.map_shared_rank(mine, c) + h * 4;
            m = fmaxf(m, st[0]);
            w = fmaxf(w, st[1]);
        }
        float v[4] = {0.f, 0.f, 0.f, 0.f};
        for (int c = 0; c < C; ++c) {
            const float* st = cluster.map_shared_rank(mine, c) + h * 4;
            l += st[2] == 0.f ? 0.f : st[0] == -INFINITY ? st[2] : st[2] * ex2(st[0] - m);
            const float f = ratio(st[1], w);
            const float4 x = *reinterpret_cast<const float4*>(cluster.map_shared_rank(o_s, c) + (size_t)h * LD + d);
            v[0] = fmaf(x.x, f, v[0]);
            v[1] = fmaf(x.y, f, v[1]);
            v[2] = fmaf(x.z, f, v[2]);
            v[3] = fmaf(x.w, f, v[3]);
        }
        // 2^(m' - m) / l: the two maxima differ by the values' exponents at most
        const float f = l == 0.f ? 0.f : ex2(w == -INFINITY ? 0.f : w - m) / l;
#pragma unroll
        for (int k = 0; k < 4; ++k) v[k] *= f;
        store4(a.out + (size_t)token * a.nq * D + (size_t)(kvh * G + h0 + h) * D + d, v);
    }
    if (C > 1) cluster.sync();                            // nobody leaves while its memory is read
}

template <int D> static int dec8_smem(int warps) { return (32 + warps * 32 + warps * 8 * (D + 4)) * (int)sizeof(float); }

template <int D> static int launch_decode(const Kv8DecodeArgs& a, int tokens, int blocks, int warps, cudaStream_t s) {
    auto kernel = kv8_decode_kernel<D>;
    if (warps < 1 || warps > dec8_most_warps<D>()) return -1;
    static bool configured[64] = {false};
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return (int)e;
    if (dev < 0 || dev >= 64) return -1;
    if (!configured[dev]) {
        e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, dec8_smem<D>(dec8_most_warps<D>()));
        if (e == cudaSuccess) e = cudaFuncSetAttribute(kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
        if (e != cudaSuccess) return (int)e;
        configured[dev] = true;
    }
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(blocks * a.nkv * a.head_groups, tokens);
    cfg.blockDim = dim3(32 * warps);
    cfg.dynamicSmemBytes = dec8_smem<D>(warps);
    cfg.stream = s;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = pdl_enabled();
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = blocks;
    attr[1].val.clusterDim.y = 1;
    attr[1].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 2;
    e = cudaLaunchKernelEx(&cfg, kernel, a);
    return e != cudaSuccess ? (int)e : launch_status();
}

// Token i is row i of q (rows q_stride apart, 16-byte aligned), out, token_req and cache_pos.  `blocks` blocks (1, 2, 4,
// 8 or 16, a cluster) of `warps` warps share the keys of a (token, kv head, 8 query heads).  Returns 0, a CUDA error
// code or -1 (shape refused).
MSTAR_API int mstar_kv8_decode(const void* q, int q_stride, void* out, const void* codes, const void* scales, int pages,
                               const int* block_table, int bt_stride, const int* token_req, const int* cache_pos,
                               int tokens, int nq, int nkv, int hd, int page_size, int window, int keep_first, float scale,
                               int blocks, int warps, void* stream) {
    if (tokens <= 0) return 0;
    if (nkv <= 0 || nq % nkv != 0 || page_size <= 0 || pages <= 0 || tokens > 65535 || blocks < 1 || blocks > 16 ||
        (blocks & (blocks - 1)) != 0 || ((uintptr_t)q & 15) != 0 || q_stride % 8 != 0 || ((uintptr_t)codes & 15) != 0 ||
        ((uintptr_t)out & 7) != 0 || (long long)pages * 2 * nkv * page_size > 0xffffffffll)
        return -1;
    const Kv8DecodeArgs a{(const bf16*)q, (bf16*)out, (const uint8_t*)codes, (const uint8_t*)scales, block_table,
                          token_req, cache_pos, q_stride, bt_stride, pages, nq, nkv, window, keep_first,
                          (nq / nkv + 7) / 8, scale * 1.4426950408889634f, page_split(page_size)};
    const cudaStream_t s = (cudaStream_t)stream;
    switch (hd) {
        case 64: return launch_decode<64>(a, tokens, blocks, warps, s);
        case 128: return launch_decode<128>(a, tokens, blocks, warps, s);
        case 256: return launch_decode<256>(a, tokens, blocks, warps, s);
        default: return -1;
    }
}
