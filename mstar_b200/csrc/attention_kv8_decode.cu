// Attention of single tokens over the 8-bit cache (format: kv8.cuh), bfloat16, head_dim 64, 128 or 256, any group of
// query heads, page sizes that are multiples of 8.
//
// The work is the cache's bytes: a token reads each of its keys and values once for up to 8 query heads, some 4 flops
// a byte and head.  So the kernel is built around having copies in flight: every warp has a ring of tiles of 32 keys
// of its own in shared memory, filled by TMA (boxes of 8 or 16 rows of a page) with the tiles after the one it works
// on, and no warp waits for another before the end.  (Loads into registers did not do: what is loaded a step ahead is
// waited for where the registers are handed on, 52 us instead of 20 for 64 requests with a window of 1,024.)  The
// products run on the tensor cores with the keys as rows, since 16 rows of queries would be mostly padding:
//   S^T [16 keys x 8 heads] += K [16 x 16] Q^T [16 x 8],   O^T [16 features x 8 heads] += V^T [16 x 16 keys] P^T.
// Which feature or key a fragment's element stands for is free as long as both operands agree.  So a thread's operands
// are runs of 16 bytes of a row: of K the features [16 t, 16 t + 16) and every 64 after them, of V [D/8 g, D/8 (g + 1))
// (lane = 4 g + t); and row g of a product is key g where g is even and g ^ 4 where it is odd, which puts the rows that
// eight neighbouring lanes read into different banks of the swizzled tiles.  V's pairs of keys are put together by byte
// permutes, P^T comes from S^T by a matrix transpose between registers (movmatrix).
//
// e4m3 is exact in float16, so both products take float16: the queries are scaled by a power of two a head (their
// largest number into [1, 2); what falls below float16's range is 2^-25 of that), the weights lie in [0, 1].  The
// rows' scales are put on the scores: a key's by a product, and a value's as an addend of the exponent, since 2^s_j *
// 2^e_j v_j = 2^(s_j + e_j) v_j.  The weights of the values' product are therefore 2^(s_j + e_j - m') with a maximum m'
// of their own, so that they use float16's range whatever the values' scales are; the normaliser's are 2^(s_j - m).
//
// The tiles of a (token, kv head) are dealt out in turn to the warps of a cluster of blocks, so that the lengths that
// are there decide the balance, not the bounds a launch was sized for.  The warps of a block are joined in shared
// memory, the blocks through distributed shared memory: one launch, no scratch memory, sums in a fixed order.
//
// Semantics are those of attention_generic.cu.  Waits are bounded; one that runs out sets the error word to 30.
#include <cooperative_groups.h>
#include <cuda_fp16.h>

#include "kv8.cuh"
#include "tma_util.cuh"

namespace cg = cooperative_groups;

struct Kv8DecodeArgs {
    const bf16* q;
    bf16* out;
    const uint8_t *codes, *scales;
    const int *block_table, *token_req, *cache_pos;
    int q_stride, bt_stride, pages, nq, nkv, window, keep_first, head_groups;
    float scale_log2e;
    PageSplit page;
    int box, stages;        // rows of a copy (8 or 16), tiles of a warp's ring
    int* error_word;
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

#define DEC8_KEYS 32     // keys of a tile
// Shared memory of a warp: `stages` tiles of keys and of values (blocks of [32 rows x at most 128 bytes], swizzled),
// then a scale pair a key, then the barriers; the outputs that the warps leave at the end lie over the tiles.
template <int D> __host__ __device__ constexpr int dec8_tile() { return DEC8_KEYS * D; }
template <int D> __host__ __device__ constexpr int dec8_stage() { return 2 * dec8_tile<D>(); }
template <int D> __host__ __device__ constexpr int dec8_ring(int stages) { return stages * (dec8_stage<D>() + DEC8_KEYS * 8 + 8); }
template <int D> __host__ __device__ constexpr int dec8_smem(int warps, int stages) {
    return 1024 + warps * dec8_ring<D>(stages) + (32 + warps * 32) * 4;
}

template <int D> __host__ __device__ constexpr int dec8_most_warps() { return D == 64 ? 16 : D == 128 ? 12 : 8; }

template <int D>
__global__ void __launch_bounds__(32 * dec8_most_warps<D>(), 1) kv8_decode_kernel(const __grid_constant__ CUtensorMap map, Kv8DecodeArgs a) {
    constexpr int KC = D / 64;             // 16-byte runs of a key row a thread takes
    constexpr int VW = D / 32;             // 4-byte words of a value row a thread takes
    constexpr int MT = D / 16;             // blocks of 16 features
    constexpr int RB = D < 128 ? D : 128;  // bytes of a row in a block of the tile
    constexpr int NB = D / RB;             // blocks of a tile
    extern __shared__ unsigned char smem_dyn[];
    unsigned char* smem8 = smem_dyn + ((1024u - (tc_smem(smem_dyn) & 1023u)) & 1023u);   // the swizzle's alignment
    pdl_wait();
    cg::cluster_group cluster = cg::this_cluster();
    const int W = blockDim.x >> 5, warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    const int C = cluster.num_blocks(), rank = cluster.block_rank(), S = a.stages;
    const int pair = blockIdx.x / C, token = blockIdx.y;
    const int kvh = pair / a.head_groups, h0 = (pair % a.head_groups) * 8, G = a.nq / a.nkv, heads = min(8, G - h0);
    const int pos = a.cache_pos[token];
    const int* bt = a.block_table + (size_t)a.token_req[token] * a.bt_stride;

    // the tiles: those of the kept first keys that lie before the window's first tile, then the window's
    const int lo = a.window > 0 ? max(0, pos - a.window + 1) : 0, first = lo / DEC8_KEYS;
    const int kept = min((min(a.keep_first, lo) + DEC8_KEYS - 1) / DEC8_KEYS, first);
    const int tiles = pos < 0 ? 0 : kept + pos / DEC8_KEYS - first + 1, stride = C * W;
    auto key0_of = [&](int i) { return (i < kept ? i : i - kept + first) * DEC8_KEYS; };

    unsigned char* ring = smem8 + (size_t)warp * S * dec8_stage<D>();
    float2* sc_s = reinterpret_cast<float2*>(smem8 + (size_t)W * S * dec8_stage<D>()) + warp * S * DEC8_KEYS;
    const uint32_t full = tc_smem(smem8 + (size_t)W * S * (dec8_stage<D>() + DEC8_KEYS * 8)) + warp * S * 8;
    if (lane < S) mbar_init(full + 8 * lane, 1);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    __syncwarp();

    // the row (of the cache as a matrix of D bytes a row) of this lane's key of a tile.  What lies past the table or on
    // pages that are not there is brought into the cache and masked.
    auto row_of = [&](int i) -> uint32_t {
        const int key = key0_of(i) + lane, logical = page_of(a.page, key);
        return ((uint32_t)page_id(bt, logical, a.bt_stride, a.pages) * 2 * a.nkv + kvh) * a.page.size +
               (uint32_t)(key - logical * a.page.size);
    };
    const uint32_t plane = (uint32_t)a.nkv * a.page.size;
    auto copy_tile = [&](int slot, uint32_t row) {
        if (lane == 0) mbar_expect_tx(full + 8 * slot, dec8_stage<D>());
        __syncwarp();
        if ((lane & (a.box - 1)) == 0) {
            const uint32_t dst = tc_smem(ring + (size_t)slot * dec8_stage<D>()) + lane * RB;
#pragma unroll
            for (int b = 0; b < NB; ++b) {
                tma_load_2d(dst + b * DEC8_KEYS * RB, &map, full + 8 * slot, b * RB, (int)row);
                tma_load_2d(dst + dec8_tile<D>() + b * DEC8_KEYS * RB, &map, full + 8 * slot, b * RB, (int)(row + plane));
            }
        }
    };
    // the scale bytes of a key and of its value, and what the softmax makes of them: 2^e and e; NaN for a bad row
    auto load_scales = [&](uint32_t row) -> uint32_t {
        return (uint32_t)a.scales[row] | ((uint32_t)a.scales[(size_t)row + plane] << 8);
    };
    auto keep_scales = [&](int slot, uint32_t two) {
        const int ks = two & 255, vs = two >> 8;
        const bool bad = ks == KV8_BAD_BYTE || vs == KV8_BAD_BYTE;
        sc_s[slot * DEC8_KEYS + lane] = make_float2(bad ? __int_as_float(0x7fc00000) : kv8_scale(ks), (float)(vs - 127));
    };

    // the ring's first tiles; from then on the tile S turns ahead is copied when its place is free, its table entry
    // being read a turn before that and its scales put into place a turn after
    const int i0 = rank * W + warp;
    uint32_t row = 0, pending = 0;
    for (int s = 0; s < S; ++s)
        if (i0 + s * stride < tiles) {
            row = row_of(i0 + s * stride);
            copy_tile(s, row);
            keep_scales(s, load_scales(row));
        }
    if (i0 + S * stride < tiles) row = row_of(i0 + S * stride);

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

    // a product's row g is key kg of its 8 (and kg + 8); a product's key 2t is key 2t, its key 2t + 1 is (2t + 1) ^ 4
    const int kg = (g & 1) ? g ^ 4 : g, kt = (2 * t + 1) ^ 4;
    // where a 16-byte run c of row r lies in a block of the tile: the swizzle of 128- or 64-byte rows
    auto at = [](int r, int c) { return r * RB + ((RB == 128 ? c ^ (r & 7) : c ^ ((r >> 1) & 3)) << 4); };
    int slot = 0;
    uint32_t parity = 0;
    int i = i0;
    for (; i < tiles; i += stride) {
        if (!__all_sync(0xffffffffu, mbar_wait(full + 8 * slot, parity))) {
            if (lane == 0) atomicExch(a.error_word, 30);
            break;
        }
        const unsigned char* kt_s = ring + (size_t)slot * dec8_stage<D>();
        const unsigned char* vt_s = kt_s + dec8_tile<D>();
        const float2* sc = sc_s + slot * DEC8_KEYS;
        const int key0 = key0_of(i);
        // ---- scores
        float s[2][4];
#pragma unroll
        for (int u = 0; u < 2; ++u) {
            s[u][0] = s[u][1] = s[u][2] = s[u][3] = 0.f;
#pragma unroll
            for (int c = 0; c < KC; ++c) {
                const unsigned char* blk = kt_s + (c >> 1) * (DEC8_KEYS * RB);
                const uint4 x = *reinterpret_cast<const uint4*>(blk + at(16 * u + kg, t + 4 * (c & 1)));
                const uint4 y = *reinterpret_cast<const uint4*>(blk + at(16 * u + kg + 8, t + 4 * (c & 1)));
                const uint32_t lo4[4] = {x.x, x.y, x.z, x.w}, hi4[4] = {y.x, y.y, y.z, y.w};
#pragma unroll
                for (int k = 0; k < 4; ++k)
                    mma_f16_16816(s[u], e4m3x2_to_f16x2(lo4[k]), e4m3x2_to_f16x2(hi4[k]), e4m3x2_hi_to_f16x2(lo4[k]),
                                  e4m3x2_hi_to_f16x2(hi4[k]), qf[c * 4 + k][0], qf[c * 4 + k][1]);
            }
        }
        // ---- weights; this thread has keys kg, kg + 8 of every 16 and heads 2t, 2t + 1
        const bool whole = key0 >= lo && key0 + DEC8_KEYS - 1 <= pos;
        float p[2][4];                       // exponents of the values' weights
        float x0 = -INFINITY, x1 = -INFINITY, y0 = -INFINITY, y1 = -INFINITY;
#pragma unroll
        for (int u = 0; u < 2; ++u)
#pragma unroll
            for (int k = 0; k < 2; ++k) {
                const int j = 16 * u + 8 * k + kg;
                const float2 f = sc[j];
                float b0 = s[u][2 * k] * f.x * hs0, b1 = s[u][2 * k + 1] * f.x * hs1;
                if (!whole) {
                    const int key = key0 + j;
                    if (key > pos || (key < lo && key >= a.keep_first)) b0 = b1 = -INFINITY;
                }
                s[u][2 * k] = b0;
                s[u][2 * k + 1] = b1;
                p[u][2 * k] = b0 + f.y;
                p[u][2 * k + 1] = b1 + f.y;
                x0 = fmaxf(x0, b0);
                x1 = fmaxf(x1, b1);
                y0 = fmaxf(y0, b0 + f.y);
                y1 = fmaxf(y1, b1 + f.y);
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
        if (__any_sync(0xffffffffu, (x0 != m0) | (x1 != m1) | (y0 != w0) | (y1 != w1))) {
            l0 *= ratio(m0, x0);
            l1 *= ratio(m1, x1);
            const float r0 = ratio(w0, y0), r1 = ratio(w1, y1);
#pragma unroll
            for (int k = 0; k < MT; ++k) {
                o[k][0] *= r0;
                o[k][1] *= r1;
                o[k][2] *= r0;
                o[k][3] *= r1;
            }
        }
        m0 = x0;
        m1 = x1;
        w0 = y0;
        w1 = y1;
        const float z0 = x0 == -INFINITY ? 0.f : x0, z1 = x1 == -INFINITY ? 0.f : x1;
        const float q0 = y0 == -INFINITY ? 0.f : y0, q1 = y1 == -INFINITY ? 0.f : y1;
        uint32_t pf[2][2];
#pragma unroll
        for (int u = 0; u < 2; ++u)
#pragma unroll
            for (int k = 0; k < 2; ++k) {
                l0 += ex2(s[u][2 * k] - z0);
                l1 += ex2(s[u][2 * k + 1] - z1);
                pf[u][k] = transpose_8x8(pack_f16(ex2(p[u][2 * k] - q0), ex2(p[u][2 * k + 1] - q1)));
            }
        // ---- values
#pragma unroll
        for (int u = 0; u < 2; ++u) {
            uint32_t v[4][VW];
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                const int r = 16 * u + 8 * (k >> 1) + ((k & 1) ? kt : 2 * t);
                if constexpr (D == 64) {
                    const uint2 w = *reinterpret_cast<const uint2*>(vt_s + at(r, g >> 1) + (g & 1) * 8);
                    v[k][0] = w.x;
                    v[k][1] = w.y;
                } else {
#pragma unroll
                    for (int c = 0; c < VW / 4; ++c) {
                        const int run = g * (VW / 4) + c;
                        const uint4 w = *reinterpret_cast<const uint4*>(vt_s + (run >> 3) * (DEC8_KEYS * RB) + at(r, run & 7));
                        v[k][4 * c] = w.x; v[k][4 * c + 1] = w.y; v[k][4 * c + 2] = w.z; v[k][4 * c + 3] = w.w;
                    }
                }
                if (!whole) {                // rows that nobody wrote may hold anything
                    const int key = key0 + r;
                    if (key > pos || (key < lo && key >= a.keep_first))
#pragma unroll
                        for (int c = 0; c < VW; ++c) v[k][c] = 0u;
                }
            }
#pragma unroll
            for (int j = 0; j < VW; ++j) {
                // features 4j, 4j + 1 and 4j + 2, 4j + 3 of this thread's run, two keys side by side
                const uint32_t a01 = __byte_perm(v[0][j], v[1][j], 0x5140), a23 = __byte_perm(v[0][j], v[1][j], 0x7362);
                const uint32_t b01 = __byte_perm(v[2][j], v[3][j], 0x5140), b23 = __byte_perm(v[2][j], v[3][j], 0x7362);
                mma_f16_16816(o[2 * j], e4m3x2_to_f16x2(a01), e4m3x2_hi_to_f16x2(a01), e4m3x2_to_f16x2(b01),
                              e4m3x2_hi_to_f16x2(b01), pf[u][0], pf[u][1]);
                mma_f16_16816(o[2 * j + 1], e4m3x2_to_f16x2(a23), e4m3x2_hi_to_f16x2(a23), e4m3x2_to_f16x2(b23),
                              e4m3x2_hi_to_f16x2(b23), pf[u][0], pf[u][1]);
            }
        }
        // ---- the tile S turns ahead takes this one's place
        __syncwarp();
        const int ahead = i + S * stride, before = slot == 0 ? S - 1 : slot - 1;
        if (i != i0 && ahead - stride < tiles) keep_scales(before, pending);
        if (ahead < tiles) {
            copy_tile(slot, row);
            pending = load_scales(row);
            if (ahead + stride < tiles) row = row_of(ahead + stride);
        }
        __syncwarp();
        if (++slot == S) {
            slot = 0;
            parity ^= 1;
        }
    }
    for (int k = 0; k < S && i < tiles; ++k, i += stride) {      // given up: not to leave before the copies under way
        mbar_wait(full + 8 * slot, parity);
        if (++slot == S) {
            slot = 0;
            parity ^= 1;
        }
    }
    pdl_launch_dependents();
    __syncthreads();

    // ---- the warps of the block: statistics (m, m', l) and outputs of 8 heads each
    constexpr int LD = D + 4;
#pragma unroll
    for (int d = 4; d < 32; d <<= 1) {
        l0 += __shfl_xor_sync(0xffffffffu, l0, d);
        l1 += __shfl_xor_sync(0xffffffffu, l1, d);
    }
    float* o_s = reinterpret_cast<float*>(smem8);         // [W][8][LD], the block's own in the first warp's place
    float* mine = reinterpret_cast<float*>(smem8 + (size_t)W * dec8_ring<D>(S));     // the block's own: [8][4]
    float* st_s = mine + 32;                              // [W][8][4]
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

template <int D>
static int launch_decode(const CUtensorMap& map, const Kv8DecodeArgs& a, int tokens, int blocks, int warps, cudaStream_t s) {
    auto kernel = kv8_decode_kernel<D>;
    const int smem = dec8_smem<D>(warps, a.stages);
    if (warps < 1 || warps > dec8_most_warps<D>() || a.stages < 2 || a.stages > 8 || smem > 227 * 1024) return -1;
    static bool configured[64] = {false};
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return (int)e;
    if (dev < 0 || dev >= 64) return -1;
    if (!configured[dev]) {
        e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, 227 * 1024);
        if (e == cudaSuccess) e = cudaFuncSetAttribute(kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
        // several blocks an SM need nearly all of its shared memory
        if (e == cudaSuccess)
            e = cudaFuncSetAttribute(kernel, cudaFuncAttributePreferredSharedMemoryCarveout, (int)cudaSharedmemCarveoutMaxShared);
        if (e != cudaSuccess) return (int)e;
        configured[dev] = true;
    }
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(blocks * a.nkv * a.head_groups, tokens);
    cfg.blockDim = dim3(32 * warps);
    cfg.dynamicSmemBytes = smem;
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
    e = cudaLaunchKernelEx(&cfg, kernel, map, a);
    return e != cudaSuccess ? (int)e : launch_status();
}

// Token i is row i of q (rows q_stride apart, 16-byte aligned), out, token_req and cache_pos.  `blocks` blocks (1, 2, 4,
// 8 or 16, a cluster) of `warps` warps with rings of `stages` tiles share the keys of a (token, kv head, 8 query heads).
// page_size: a multiple of 8.  Returns 0, a CUDA error code or -1 (shape refused).
MSTAR_API int mstar_kv8_decode(const void* q, int q_stride, void* out, const void* codes, const void* scales, int pages,
                               const int* block_table, int bt_stride, const int* token_req, const int* cache_pos,
                               int tokens, int nq, int nkv, int hd, int page_size, int window, int keep_first, float scale,
                               int blocks, int warps, int stages, int* error_word, void* stream) {
    if (tokens <= 0) return 0;
    const long long rows = (long long)pages * 2 * nkv * page_size;
    if (nkv <= 0 || nq % nkv != 0 || page_size <= 0 || page_size % 8 != 0 || pages <= 0 || tokens > 65535 || blocks < 1 ||
        blocks > 16 || (blocks & (blocks - 1)) != 0 || ((uintptr_t)q & 15) != 0 || q_stride % 8 != 0 ||
        ((uintptr_t)codes & 15) != 0 || ((uintptr_t)out & 7) != 0 || rows > 0x7fffffffll || error_word == nullptr ||
        (hd != 64 && hd != 128 && hd != 256))
        return -1;
    const int box = page_size % 16 == 0 ? 16 : 8;
    // the cache as a matrix of `rows` rows of hd bytes
    CUtensorMap map;
    {
        EncodeTiledFn encode = encode_tiled_fn();
        if (encode == nullptr) return (int)cudaErrorNotSupported;
        const cuuint64_t dims[2] = {(cuuint64_t)hd, (cuuint64_t)rows};
        const cuuint64_t strides[1] = {(cuuint64_t)hd};
        const cuuint32_t size[2] = {(cuuint32_t)(hd < 128 ? hd : 128), (cuuint32_t)box};
        const cuuint32_t elem[2] = {1, 1};
        if (encode(&map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<void*>(codes), dims, strides, size, elem,
                   CU_TENSOR_MAP_INTERLEAVE_NONE, hd < 128 ? CU_TENSOR_MAP_SWIZZLE_64B : CU_TENSOR_MAP_SWIZZLE_128B,
                   CU_TENSOR_MAP_L2_PROMOTION_L2_128B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) != CUDA_SUCCESS)
            return -1;
    }
    const Kv8DecodeArgs a{(const bf16*)q, (bf16*)out, (const uint8_t*)codes, (const uint8_t*)scales, block_table,
                          token_req, cache_pos, q_stride, bt_stride, pages, nq, nkv, window, keep_first,
                          (nq / nkv + 7) / 8, scale * 1.4426950408889634f, page_split(page_size), box, stages, error_word};
    const cudaStream_t s = (cudaStream_t)stream;
    switch (hd) {
        case 64: return launch_decode<64>(map, a, tokens, blocks, warps, s);
        case 128: return launch_decode<128>(map, a, tokens, blocks, warps, s);
        default: return launch_decode<256>(map, a, tokens, blocks, warps, s);
    }
}
