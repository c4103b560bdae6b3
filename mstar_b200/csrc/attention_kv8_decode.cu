// Attention of single tokens over the 8-bit cache (format: kv8.cuh), bfloat16, head_dim 64, 128 or 256, any group of
// query heads, page sizes that are multiples of 8.
//
// The work is the cache's bytes: a token reads each of its keys and values once for up to 8 query heads, some 4 flops
// a byte and head.  So the kernel is built around having copies in flight: every warp has a ring of tiles of 32 keys
// of its own in shared memory, filled by asynchronous copies of 16 bytes a thread with the tiles after the one it works
// on, and no warp waits for another before the end.  (TMA boxes of a page's rows took some 700 clocks a tile to issue
// from one thread and 800 from several, against 350: 18.0 us for one token on 16,384 keys where these take 15.2.  Loads
// into registers a step ahead are waited for where the registers are handed on: 52 us for 64 requests with a window of
// 1,024 keys against 17.6.)  The products run on the tensor cores with the keys as rows, since 16 rows of queries would be mostly padding:
//   S^T [16 keys x 8 heads] += K [16 x 16] Q^T [16 x 8],   O^T [16 features x 8 heads] += V^T [16 x 16 keys] P^T.
// Which feature or key a fragment's element stands for is free as long as both operands agree.  So a thread's operands
// are runs of 16 bytes of a row: of K the features [16 t, 16 t + 16) and every 64 after them, of V [D/8 g, D/8 (g + 1))
// (lane = 4 g + t); and row g of a product is key g where g is even and g ^ 4 where it is odd, which puts the rows that
// eight neighbouring lanes read into different banks of the swizzled tiles.  V's pairs of keys are put together by byte
// permutes, P^T comes from S^T by a matrix transpose between registers (movmatrix).
//
// The scores' product takes the keys' codes as they are (e4m3 x e4m3).  A query is its largest number's power of two
// times two codes, x = hi + lo / 32: the first rounding leaves 2^-4 of a number, the second 2^-22 of the head's largest
// (a bfloat16 has 8 bits, which two codes hold but for numbers 2^-10 below the largest).  That costs a second product,
// which takes 4.6 clocks where the float16 one with half the depth takes 8 and its operands' conversion as long; with up
// to 4 query heads a kv head there is none: hi and lo are columns 0 - 3 and 4 - 7 of one product, and the threads that
// would have idle columns take half of the keys of the softmax.
//
// The rows' scales are put on the scores: a key's by a product, and a value's as an addend of the exponent, since 2^s_j *
// 2^e_j v_j = 2^(s_j + e_j) v_j.  The values' weights are therefore 2^(s_j + e_j - m') with a maximum m' of their own, the
// normaliser's 2^(s_j - m).  Both maxima follow the scores only when these exceed them by more than 2^8, which a vote of
// the warp finds: exchanging the maxima at every tile costs as much as its exponentials.
//
// The values' product is one of bfloat16, codes as they are and weights in two parts (16 bits, down to 2^-126 of the
// largest), so that a key of a small weight, or of small values beside one of large values, counts in the features where
// the large ones have zeros.  With up to 4 query heads a kv head the low parts are columns 4 - 7 of the same product, otherwise
// they take one of their own.  A code becomes a bfloat16 by moving its sign, exponent and mantissa, three to four
// instructions for two of them.  (Float16 weights, and codes by a conversion each, took 15.1 us for one token on 16,384
// keys instead of 16.8 and 41.7 for 64 on 800 to 2,048 instead of 48, but float16 ends at 2^-24, so that what lies further
// below the largest was lost in every feature.  Float16 only for tiles whose weights all allow it, found by a vote: 17.3 and 47.)
//
// The tiles of a (token, kv head) are dealt out in turn to the warps of a cluster of blocks, so that the lengths that
// are there decide the balance, not the bounds a launch was sized for.  The warps of a block are joined in shared
// memory; the blocks send what each other block is to join into its shared memory (stores that nobody waits for, then
// one barrier; reading it from there took 4,100 clocks, a wait for every block in turn): one launch, no scratch
// memory, sums in a fixed order.
//
// A warp's ring is two tiles, so that twelve warps of head_dim 128 fit an SM instead of eight (sixteen of 64): its
// instructions, issued in order and each waiting for the last, bound it, not the copies.  64 requests, 8 kv heads of 128:
// 51.1 us on 2,048 keys each (41.5 at the copy bandwidth), 48.2 on 800 to 2,048 (29.5); one on 16,384: 16.8 (5.2); 64 on
// windows of 1,024 keys of 64: 20.2 (10.6).
//
// Semantics are those of attention_generic.cu.
#include <cooperative_groups.h>

#include "kv8.cuh"
#include "mma_util.cuh"

namespace cg = cooperative_groups;

struct Kv8DecodeArgs {
    const bf16* q;
    bf16* out;
    const uint8_t *codes, *scales;
    const int *block_table, *token_req, *cache_pos;
    int q_stride, bt_stride, bt_width, pages, nq, nkv, window, keep_first, head_groups;
    float scale_log2e;
    PageSplit page;
};

// Of a word of four codes, two of each of two keys, the second or the first of both as bfloat16 times 2^-120: sign, exponent
// and mantissa in bfloat16's places (subnormal codes become subnormal numbers).
__device__ __forceinline__ uint32_t codes_second(uint32_t x) { return (x & 0x80008000u) | ((x >> 4) & 0x07f007f0u); }
__device__ __forceinline__ uint32_t codes_first(uint32_t x) { return ((x << 8) & 0x80008000u) | ((x << 4) & 0x07f007f0u); }
__device__ __forceinline__ void mma_e4m3_16832(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,
                                               uint32_t b0, uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k32.row.col.f32.e4m3.e4m3.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};\n"
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
__device__ __forceinline__ void cluster_arrive() { asm volatile("barrier.cluster.arrive.release;" ::: "memory"); }
__device__ __forceinline__ void cluster_wait() { asm volatile("barrier.cluster.wait.acquire;" ::: "memory"); }
// 2^(a - b) for maxima that may still be -inf (of a part without keys: 0)
__device__ __forceinline__ float ratio(float a, float b) { return a == -INFINITY ? 0.f : ex2(a - b); }

#define DEC8_KEYS 32     // keys of a tile
#define DEC8_STAGES 2    // tiles of a warp's ring
#define DEC8_SLACK 8.f   // how far (in powers of two) scores may exceed the maxima
#define DEC8_RAISE 112.f // weights are at most 2^(112 + 8)
// Shared memory of a warp: tiles of keys and of values (blocks of [32 rows x at most 128 bytes], swizzled), then a scale
// pair a key, then each tile's scale bytes; the outputs that the warps leave at the end lie over the tiles.
template <int D> __host__ __device__ constexpr int dec8_tile() { return DEC8_KEYS * D; }
template <int D> __host__ __device__ constexpr int dec8_stage() { return 2 * dec8_tile<D>() + 2 * DEC8_KEYS; }
template <int D> __host__ __device__ constexpr int dec8_ring() { return DEC8_STAGES * dec8_stage<D>() + DEC8_KEYS * 8; }
// Of a block: the warps' statistics, the blocks' statistics [8][8][4], and a place for the parts of all blocks of what
// this block joins, [C][H][D / C].
template <int D, int H> __host__ __device__ constexpr int dec8_smem(int warps, int blocks) {
    return warps * dec8_ring<D>() + (warps * 32 + (blocks > 1 ? 8 * 32 + H * D : 0)) * 4;
}
template <int D> __host__ __device__ constexpr int dec8_most_warps() { return D == 64 ? 16 : D == 128 ? 8 : 4; }

// H: query heads of a block, 4 or 8
template <int D, int H>
__global__ void __launch_bounds__(32 * dec8_most_warps<D>(), 1)
kv8_decode_kernel(Kv8DecodeArgs a) {
    constexpr int KC = D / 64;             // 16-byte runs of a key row a thread takes
    constexpr int VW = D / 32;             // 4-byte words of a value row a thread takes
    constexpr int MT = D / 16;             // blocks of 16 features
    constexpr int RB = D < 128 ? D : 128;  // bytes of a row in a block of the tile
    constexpr int S = DEC8_STAGES;
    constexpr int E = H == 4 ? 1 : 2;      // keys of every 16 whose weights a thread makes, for two heads each
    extern __shared__ __align__(1024) unsigned char smem8[];
    const int W = blockDim.x >> 5, warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    // the tiles of all warps lie first, then the rest, so that the tiles keep their alignment
    unsigned char* ring = smem8 + (size_t)warp * S * 2 * dec8_tile<D>();
    float2* sc = reinterpret_cast<float2*>(smem8 + (size_t)W * S * 2 * dec8_tile<D>()) + warp * DEC8_KEYS;
    unsigned char* bytes_s = smem8 + (size_t)W * (S * 2 * dec8_tile<D>() + DEC8_KEYS * 8) + warp * S * 2 * DEC8_KEYS;
    cluster_arrive();                       // (everybody has started before anybody's memory is written)
    pdl_wait();
    cg::cluster_group cluster = cg::this_cluster();
    const int C = cluster.num_blocks(), rank = cluster.block_rank();
    const int pair = blockIdx.x / C, token = blockIdx.y;
    const int pos = a.cache_pos[token];
    const int* bt = a.block_table + (size_t)a.token_req[token] * a.bt_stride;
    const int kvh = pair / a.head_groups, h0 = (pair % a.head_groups) * H, G = a.nq / a.nkv, heads = min(H, G - h0);

    // this thread's part of a query (head g, with H = 4 head g % 4): the features that its part of K has
    uint32_t raw[KC][8];
    const int qh = H == 4 ? g & 3 : g;
    {
        const bf16* q = a.q + (size_t)token * a.q_stride + (size_t)(kvh * G + h0 + (qh < heads ? qh : 0)) * D;
#pragma unroll
        for (int c = 0; c < KC; ++c)
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                const uint4 w = *reinterpret_cast<const uint4*>(q + c * 64 + t * 16 + i * 8);
                raw[c][4 * i] = w.x; raw[c][4 * i + 1] = w.y; raw[c][4 * i + 2] = w.z; raw[c][4 * i + 3] = w.w;
            }
    }

    // the tiles: those of the kept first keys that lie before the window's first tile, then the window's
    const int lo = a.window > 0 ? max(0, pos - a.window + 1) : 0, first = lo / DEC8_KEYS;
    const int kept = min((min(a.keep_first, lo) + DEC8_KEYS - 1) / DEC8_KEYS, first);
    const int tiles = pos < 0 ? 0 : kept + pos / DEC8_KEYS - first + 1, stride = C * W;
    auto key0_of = [&](int i) { return (i < kept ? i : i - kept + first) * DEC8_KEYS; };
    // The row (of the cache as a matrix of D bytes a row) of this lane's key of a tile, from the table's entry for it.
    // What lies past the table or on pages that are not there is brought into the cache and masked.  (Two steps: a warp
    // issues in order, and would stand still at the first use of an entry just asked for.)
    auto entry_of = [&](int i) -> int { return bt[min(page_of(a.page, key0_of(i) + lane), a.bt_width - 1)]; };
    auto row_of = [&](int i, int entry) -> uint32_t {
        const int key = key0_of(i) + lane, page = (int)min((unsigned)entry, (unsigned)(a.pages - 1));
        return ((uint32_t)page * 2 * a.nkv + kvh) * a.page.size + (uint32_t)(key - page_of(a.page, key) * a.page.size);
    };
    const uint32_t plane = (uint32_t)a.nkv * a.page.size;
    // where a 16-byte run c of row r lies in a block of the tile: the swizzle of 128- or 64-byte rows
    auto at = [](int r, int c) { return r * RB + ((RB == 128 ? c ^ (r & 7) : c ^ ((r >> 1) & 3)) << 4); };
    // starts the copies of a tile; `row`: of this lane's key.  Groups of 8 keys lie in one page, their scale bytes side
    // by side.  Always one group of copies, so that they can be counted.
    auto copy_tile = [&](int slot, uint32_t row, bool there) {
        if (there) {
            constexpr int CPR = D / 16, RPI = 32 / CPR;       // 16-byte runs of a row, rows of a warp's copy
            const uint32_t dst = smem_u32(ring) + slot * 2 * dec8_tile<D>();
            const int run = lane % CPR;
            // (all rows first: copies keep their order, and an exchange between two of them would be waited for)
            const uint8_t* src[DEC8_KEYS / RPI];
#pragma unroll
            for (int k = 0; k < DEC8_KEYS / RPI; ++k)
                src[k] = a.codes + (size_t)__shfl_sync(0xffffffffu, row, k * RPI + lane / CPR) * D + run * 16;
#pragma unroll
            for (int k = 0; k < DEC8_KEYS / RPI; ++k) {
                const uint32_t to = dst + (run >> 3) * (DEC8_KEYS * RB) + at(k * RPI + lane / CPR, run & 7);
                cp_async_16(to, src[k], 16);
                cp_async_16(to + dec8_tile<D>(), src[k] + (size_t)plane * D, 16);
            }
            if ((lane & 7) == 0) {
                const uint32_t to = smem_u32(bytes_s) + slot * 2 * DEC8_KEYS + lane;
                cp_async_8(to, a.scales + row);
                cp_async_8(to + DEC8_KEYS, a.scales + (size_t)row + plane);
            }
        }
        cp_async_commit();
    };

    // the table's entries of the ring's first tiles; they come while the queries are made ready
    const int i0 = rank * W + warp;
    int entry = 0, entries[S];
#pragma unroll
    for (int s = 0; s < S; ++s) entries[s] = i0 + s * stride < tiles ? entry_of(i0 + s * stride) : 0;
    if (i0 + S * stride < tiles) entry = entry_of(i0 + S * stride);

    // the query's codes: hi and lo (with H = 4 in the threads of g < 4 and of g >= 4)
    uint32_t qf[H == 4 ? 1 : 2][4 * KC];
    float head_scale;
    {
        float most = 0.f;
#pragma unroll
        for (int c = 0; c < KC; ++c)
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                if (qh >= heads) raw[c][i] = 0u;
                const float2 f = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&raw[c][i]));
                most = fabsf(f.x) < INFINITY && fabsf(f.y) < INFINITY ? fmaxf(most, fmaxf(fabsf(f.x), fabsf(f.y))) : INFINITY;
            }
        most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, 1));
        most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, 2));
        // the largest number into [128, 256); a query that is not finite gives NaNs
        const uint32_t e = max(__float_as_uint(most) >> 23, 8u);
        const float down = e < 255u ? __uint_as_float((261u - e) << 23) : 1.f;
        head_scale = e < 255u ? __uint_as_float((e - 7u) << 23) * a.scale_log2e : __int_as_float(0x7fc00000);
#pragma unroll
        for (int c = 0; c < KC; ++c)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const float2 x = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&raw[c][2 * i]));
                const float2 y = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&raw[c][2 * i + 1]));
                const float v[4] = {x.x * down, x.y * down, y.x * down, y.y * down};
                const uint32_t hi = kv8_pack4(v[0], v[1], v[2], v[3]);
                float r[4];
                kv8_unpack4(hi, r);
                const uint32_t rest = kv8_pack4((v[0] - r[0]) * 32.f, (v[1] - r[1]) * 32.f, (v[2] - r[2]) * 32.f, (v[3] - r[3]) * 32.f);
                if constexpr (H == 4) {
                    qf[0][4 * c + i] = g < 4 ? hi : rest;
                } else {
                    qf[0][4 * c + i] = hi;
                    qf[H == 4 ? 0 : 1][4 * c + i] = rest;
                }
            }
    }
    // of the two heads whose scores this thread has: 2t, 2t + 1, with H = 4 2 (t % 2) and the next
    const int th = H == 4 ? t & 1 : t;
    const float hs0 = __shfl_sync(0xffffffffu, head_scale, 8 * th), hs1 = __shfl_sync(0xffffffffu, head_scale, 8 * th + 4);

    // the ring's first tiles; from then on the tile S turns ahead is copied when its place is free, its table entry
    // having been read a turn before
#pragma unroll
    for (int s = 0; s < S; ++s) copy_tile(s, row_of(i0 + s * stride, entries[s]), i0 + s * stride < tiles);

    float o[MT][4];
#pragma unroll
    for (int i = 0; i < MT; ++i) o[i][0] = o[i][1] = o[i][2] = o[i][3] = 0.f;
    float m0 = -INFINITY, m1 = -INFINITY, w0 = -INFINITY, w1 = -INFINITY, l0 = 0.f, l1 = 0.f;

    // a product's row g is key kg of its 8 (and kg + 8); a product's key 2t is key 2t, its key 2t + 1 is (2t + 1) ^ 4
    const int kg = (g & 1) ? g ^ 4 : g, kt = (2 * t + 1) ^ 4;
    const int kmine = kg + (H == 4 && t >= 2 ? 8 : 0);        // the first key of 16 whose weights this thread makes
    int slot = 0;
    for (int i = i0; i < tiles; i += stride) {
        cp_async_wait<S - 1>();
        __syncwarp();
        const unsigned char* kt_s = ring + slot * 2 * dec8_tile<D>();
        const unsigned char* vt_s = kt_s + dec8_tile<D>();
        // a lane makes its key's scales ready: 2^e of the key (NaN for a bad row) and e of the value
        {
            const int ks = bytes_s[slot * 2 * DEC8_KEYS + lane], vs = bytes_s[(slot * 2 + 1) * DEC8_KEYS + lane];
            const bool bad = ks == KV8_BAD_BYTE || vs == KV8_BAD_BYTE;
            sc[lane] = make_float2(bad ? __int_as_float(0x7fc00000) : kv8_scale(ks), (float)(vs - 127));
        }
        const int key0 = key0_of(i);
        // ---- scores: s[u][2k + h] of the thread's k-th key of 16 and its h-th head
        float s[2][2 * E];
        {
            // (sums of hi and of lo products; all products before the exchanges, which would wait for theirs in turn)
            float x[2][4], y[2][4];
#pragma unroll
            for (int u = 0; u < 2; ++u)
#pragma unroll
                for (int k = 0; k < 4; ++k) x[u][k] = y[u][k] = 0.f;
#pragma unroll
            for (int c = 0; c < KC; ++c)
#pragma unroll
                for (int u = 0; u < 2; ++u) {
                    const unsigned char* blk = kt_s + (c >> 1) * (DEC8_KEYS * RB);
                    const uint4 ka = *reinterpret_cast<const uint4*>(blk + at(16 * u + kg, t + 4 * (c & 1)));
                    const uint4 kb = *reinterpret_cast<const uint4*>(blk + at(16 * u + kg + 8, t + 4 * (c & 1)));
                    if constexpr (H == 4) {
                        mma_e4m3_16832(x[u], ka.x, kb.x, ka.y, kb.y, qf[0][4 * c], qf[0][4 * c + 1]);
                        mma_e4m3_16832(y[u], ka.z, kb.z, ka.w, kb.w, qf[0][4 * c + 2], qf[0][4 * c + 3]);
                    } else {
                        mma_e4m3_16832(x[u], ka.x, kb.x, ka.y, kb.y, qf[0][4 * c], qf[0][4 * c + 1]);
                        mma_e4m3_16832(y[u], ka.x, kb.x, ka.y, kb.y, qf[1][4 * c], qf[1][4 * c + 1]);
                        mma_e4m3_16832(x[u], ka.z, kb.z, ka.w, kb.w, qf[0][4 * c + 2], qf[0][4 * c + 3]);
                        mma_e4m3_16832(y[u], ka.z, kb.z, ka.w, kb.w, qf[1][4 * c + 2], qf[1][4 * c + 3]);
                    }
                }
            if constexpr (H == 4) {
                // threads of t < 2 have the hi sums, the others the lo sums; the former keep key kg, the latter kg + 8
                float got[2][2];
#pragma unroll
                for (int u = 0; u < 2; ++u)
#pragma unroll
                    for (int k = 0; k < 4; ++k) x[u][k] += y[u][k];
#pragma unroll
                for (int u = 0; u < 2; ++u)
#pragma unroll
                    for (int h = 0; h < 2; ++h) got[u][h] = __shfl_xor_sync(0xffffffffu, t < 2 ? x[u][2 + h] : x[u][h], 2);
#pragma unroll
                for (int u = 0; u < 2; ++u)
#pragma unroll
                    for (int h = 0; h < 2; ++h)
                        s[u][h] = t < 2 ? fmaf(got[u][h], 0.03125f, x[u][h]) : fmaf(x[u][2 + h], 0.03125f, got[u][h]);
            } else {
#pragma unroll
                for (int u = 0; u < 2; ++u)
#pragma unroll
                    for (int k = 0; k < 4; ++k) s[u][k] = fmaf(y[u][k], 0.03125f, x[u][k]);
            }
        }
        // ---- weights
        __syncwarp();
        const bool whole = key0 >= lo && key0 + DEC8_KEYS - 1 <= pos;
        float p[2][2 * E];                   // exponents of the values' weights
        float x0 = -INFINITY, x1 = -INFINITY, y0 = -INFINITY, y1 = -INFINITY;
#pragma unroll
        for (int u = 0; u < 2; ++u)
#pragma unroll
            for (int k = 0; k < E; ++k) {
                const int j = 16 * u + 8 * k + kmine;
                const float2 f = sc[j];
                float b0 = s[u][2 * k] * (f.x * hs0), b1 = s[u][2 * k + 1] * (f.x * hs1);
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
        // (a maximum is -inf only where every score so far is NaN or -inf: the sums are NaN or zero then)
        if (__any_sync(0xffffffffu, (x0 > m0 + DEC8_SLACK) | (x1 > m1 + DEC8_SLACK) | (y0 > w0 + DEC8_SLACK) |
                                        (y1 > w1 + DEC8_SLACK))) {
#pragma unroll
            for (int d = H == 4 ? 2 : 4; d < 32; d <<= 1) {
                x0 = fmaxf(x0, __shfl_xor_sync(0xffffffffu, x0, d));
                x1 = fmaxf(x1, __shfl_xor_sync(0xffffffffu, x1, d));
                y0 = fmaxf(y0, __shfl_xor_sync(0xffffffffu, y0, d));
                y1 = fmaxf(y1, __shfl_xor_sync(0xffffffffu, y1, d));
            }
            x0 = fmaxf(m0, x0);
            x1 = fmaxf(m1, x1);
            y0 = fmaxf(w0, y0);
            y1 = fmaxf(w1, y1);
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
            m0 = x0;
            m1 = x1;
            w0 = y0;
            w1 = y1;
        }
        const float z0 = m0 == -INFINITY ? 0.f : m0, z1 = m1 == -INFINITY ? 0.f : m1;
        // (the weights' exponents are raised so that the products with codes times 2^-120 are as large as they would be without)
        const float q0 = (w0 == -INFINITY ? 0.f : w0) - DEC8_RAISE, q1 = (w1 == -INFINITY ? 0.f : w1) - DEC8_RAISE;
        uint32_t pf[2][2], pl[2][2];          // the weights' bfloat16 parts
#pragma unroll
        for (int u = 0; u < 2; ++u)
#pragma unroll
            for (int k = 0; k < E; ++k) {
                l0 += ex2(s[u][2 * k] - z0);
                l1 += ex2(s[u][2 * k + 1] - z1);
                const float p0 = ex2(p[u][2 * k] - q0), p1 = ex2(p[u][2 * k + 1] - q1);
                const uint32_t hi = pack_bf16(p0, p1);
                pf[u][k] = transpose_8x8(hi);
                pl[u][k] = transpose_8x8(pack_bf16(p0 - __uint_as_float(hi << 16), p1 - __uint_as_float(hi & 0xffff0000u)));
            }
        if constexpr (H == 4) {
            // row g < 4 of a transpose is head g with the first eight keys, row g + 4 the same head with the others: columns
            // 0 - 3 of the product take the high parts of both, columns 4 - 7 the low ones
#pragma unroll
            for (int u = 0; u < 2; ++u) {
                const uint32_t got = __shfl_xor_sync(0xffffffffu, g < 4 ? pl[u][0] : pf[u][0], 16);
                pf[u][1] = g < 4 ? got : pl[u][0];
                pf[u][0] = g < 4 ? pf[u][0] : got;
            }
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
                // features 4j, 4j + 1 and 4j + 2, 4j + 3 of this thread's run, of one key and of the other
                const uint32_t a01 = __byte_perm(v[0][j], v[1][j], 0x5410), a23 = __byte_perm(v[0][j], v[1][j], 0x7632);
                const uint32_t b01 = __byte_perm(v[2][j], v[3][j], 0x5410), b23 = __byte_perm(v[2][j], v[3][j], 0x7632);
                const uint32_t lo[4] = {codes_first(a01), codes_second(a01), codes_first(b01), codes_second(b01)};
                const uint32_t hi[4] = {codes_first(a23), codes_second(a23), codes_first(b23), codes_second(b23)};
                if constexpr (H == 8) {
                    mma_bf16_16816(o[2 * j], lo, pl[u][0], pl[u][1]);
                    mma_bf16_16816(o[2 * j + 1], hi, pl[u][0], pl[u][1]);
                }
                mma_bf16_16816(o[2 * j], lo, pf[u][0], pf[u][1]);
                mma_bf16_16816(o[2 * j + 1], hi, pf[u][0], pf[u][1]);
            }
        }
        // ---- the tile S turns ahead takes this one's place
        __syncwarp();
        const int ahead = i + S * stride;
        copy_tile(slot, row_of(ahead, entry), ahead < tiles);
        if (ahead + stride < tiles) entry = entry_of(ahead + stride);
        if (++slot == S) slot = 0;
    }
    cp_async_wait<0>();
    pdl_launch_dependents();
    __syncthreads();

    // ---- the warps of the block: statistics (m, m', l) and outputs of H heads each
    if constexpr (H == 4) {                  // the sums of the high and of the low parts
#pragma unroll
        for (int k = 0; k < MT; ++k)
#pragma unroll
            for (int i = 0; i < 4; ++i) o[k][i] += __shfl_xor_sync(0xffffffffu, o[k][i], 2);
    }
    constexpr int LD = D + 4;
#pragma unroll
    for (int d = H == 4 ? 2 : 4; d < 32; d <<= 1) {
        l0 += __shfl_xor_sync(0xffffffffu, l0, d);
        l1 += __shfl_xor_sync(0xffffffffu, l1, d);
    }
    float* o_s = reinterpret_cast<float*>(smem8);         // [W][H][LD]
    float4* st_s = reinterpret_cast<float4*>(smem8 + (size_t)W * dec8_ring<D>());     // [W][8]
    float4* all_st = st_s + W * 8;                        // [C][8]: of the blocks
    float* all_o = reinterpret_cast<float*>(all_st + 8 * 8);
    if (g == 0 && 2 * t < H) {
        st_s[warp * 8 + 2 * t] = make_float4(m0, w0, l0, 0.f);
        st_s[warp * 8 + 2 * t + 1] = make_float4(m1, w1, l1, 0.f);
    }
    if (2 * t < H) {
        float* dst = o_s + (size_t)(warp * H + 2 * t) * LD;
#pragma unroll
        for (int k = 0; k < MT; ++k) {
            const int d = g * (D / 8) + 2 * k;            // rows g and g + 8 of the block: two neighbouring features
            *reinterpret_cast<float2*>(dst + d) = make_float2(o[k][0], o[k][2]);
            *reinterpret_cast<float2*>(dst + LD + d) = make_float2(o[k][1], o[k][3]);
        }
    }
    __syncthreads();
    // (m, m', l) of `n` parts together; a part whose every score was NaN has the maximum -inf and a sum of NaN
    auto join = [](const float4* st, int n) -> float4 {
        float m = -INFINITY, w = -INFINITY, l = 0.f;
#pragma unroll 4
        for (int k = 0; k < n; ++k) {
            m = fmaxf(m, st[k * 8].x);
            w = fmaxf(w, st[k * 8].y);
        }
#pragma unroll 4
        for (int k = 0; k < n; ++k) {
            const float4 x = st[k * 8];
            l = fmaf(x.z, x.x == -INFINITY ? 1.f : ex2(x.x - m), l);      // (x.z is 0 or NaN where x.x is -inf)
        }
        return make_float4(m, w, l, 0.f);
    };
    // sum of 2^(m'_k - w) x_k over `n` parts' four features
    auto add = [](const float4* st, const float* x, int step, int n, float w) -> float4 {
        float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 4
        for (int k = 0; k < n; ++k) {
            const float f = ratio(st[k * 8].y, w);
            const float4 y = *reinterpret_cast<const float4*>(x + (size_t)k * step);
            v.x = fmaf(y.x, f, v.x);
            v.y = fmaf(y.y, f, v.y);
            v.z = fmaf(y.z, f, v.z);
            v.w = fmaf(y.w, f, v.w);
        }
        return v;
    };
    auto finish = [&](const float4& all, const float4& v, int h, int d) {
        // 2^(m' - m) / l: the two maxima differ by the values' exponents and the slack at most.  (Sums are 2^(DEC8_RAISE - 120)
        // times what they stand for; that factor by itself, since 2^(m' - m) may be as large as 2^127.)
        const float f = all.z == 0.f ? 0.f : ex2(all.y == -INFINITY ? 0.f : all.y - all.x) / all.z;
        const float out[4] = {v.x * f * 256.f, v.y * f * 256.f, v.z * f * 256.f, v.w * f * 256.f};
        store4(a.out + (size_t)token * a.nq * D + (size_t)(kvh * G + h0 + h) * D + d, out);
    };
    // four features a thread; block c joins the features [c D / C, (c + 1) D / C) of every head
    constexpr int Q = D / 4;
    const int log_c = 31 - __clz(C), q_share = Q >> log_c;
    if (C > 1) {
        cluster_wait();
        for (int k = blockDim.x - 1 - threadIdx.x; k < heads * C; k += blockDim.x)
            *cluster.map_shared_rank(all_st + rank * 8 + (k >> log_c), k & (C - 1)) = join(st_s + (k >> log_c), W);
    }
    for (int k = threadIdx.x; k < heads * Q; k += blockDim.x) {
        const int h = k / Q, q = k % Q;
        if (C == 1) {
            const float4 all = join(st_s + h, W);
            finish(all, add(st_s + h, o_s + (size_t)h * LD + q * 4, H * LD, W, all.y), h, q * 4);
        } else {
            float w = -INFINITY;
#pragma unroll 4
            for (int i = 0; i < W; ++i) w = fmaxf(w, st_s[i * 8 + h].y);
            const int c = q / q_share;
            float4* to = reinterpret_cast<float4*>(all_o) + (rank * H + h) * q_share + (q - c * q_share);
            *cluster.map_shared_rank(to, c) = add(st_s + h, o_s + (size_t)h * LD + q * 4, H * LD, W, w);
        }
    }
    if (C == 1) {
        cluster_wait();
        return;
    }
    // ---- the blocks of the cluster: each joins its share
    cluster_arrive();
    cluster_wait();
    for (int k = threadIdx.x; k < heads * q_share; k += blockDim.x) {
        const int h = k / q_share, q = k - h * q_share;
        const float4 all = join(all_st + h, C);
        finish(all, add(all_st + h, all_o + (size_t)(h * q_share + q) * 4, H * q_share * 4, C, all.y), h,
               (rank * q_share + q) * 4);
    }
}

template <int D, int H>
static int launch_decode(const Kv8DecodeArgs& a, int tokens, int blocks, int warps, cudaStream_t s) {
    auto kernel = kv8_decode_kernel<D, H>;
    int smem = dec8_smem<D, H>(warps, blocks);
    if (warps < 1 || warps > dec8_most_warps<D>() || smem > 227 * 1024) return -1;
    static bool configured[64] = {false};
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return (int)e;
    if (dev < 0 || dev >= 64) return -1;
    if (!configured[dev]) {
        e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, 227 * 1024);
        // several blocks an SM need nearly all of its shared memory
        if (e == cudaSuccess)
            e = cudaFuncSetAttribute(kernel, cudaFuncAttributePreferredSharedMemoryCarveout, (int)cudaSharedmemCarveoutMaxShared);
        if (e != cudaSuccess) return (int)e;
        configured[dev] = true;
    }
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(blocks * a.nkv * a.head_groups, tokens);
    // No more blocks an SM than an even share, by asking for so much shared memory that one more does not fit (an SM has 228
    // KB, of which a block takes 1 KB besides; 128 bytes to spare): with room for more, some SMs take them and others none
    // (heads of 64, 2,048 keys, 32, 96, 192 pairs: 5.8, 9.5, 16.3 us so, 6.8, 10.7, 17.5 without).  Clusters of eight do not
    // fill the groups of SMs that they have to lie in, so that their share is counted over ten thirteenths of the SMs
    // (16 pairs of heads of 64 and of 128: 5.9 and 7.9 us so, 9.1 and 13.3 over all).
    const long long all = (long long)cfg.gridDim.x * tokens * (blocks >= 8 ? 13 : 10) / 10;
    const long long share = (all + device_sm_count() - 1) / device_sm_count();
    smem = max(smem, (int)min(227ll * 1024, 228 * 1024 / (share + 1) - 896));
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
    e = cudaLaunchKernelEx(&cfg, kernel, a);
    return e != cudaSuccess ? (int)e : launch_status();
}

// Token i is row i of q (rows q_stride apart, 16-byte aligned), out, token_req and cache_pos.  `blocks` blocks (1, 2, 4
// or 8, a cluster) of `warps` warps share the keys of a (token, kv head, 8 query heads, or up to 4 where a kv head has
// no more).  page_size: a multiple of 8.  Returns 0, a CUDA error code or -1 (shape refused).
MSTAR_API int mstar_kv8_decode(const void* q, int q_stride, void* out, const void* codes, const void* scales, int pages,
                               const int* block_table, int bt_stride, int bt_width, const int* token_req, const int* cache_pos,
                               int tokens, int nq, int nkv, int hd, int page_size, int window, int keep_first, float scale,
                               int blocks, int warps, void* stream) {
    if (tokens <= 0) return 0;
    if (nkv <= 0 || nq % nkv != 0 || page_size <= 0 || page_size % 8 != 0 || pages <= 0 || bt_width <= 0 ||
        tokens > 65535 || blocks < 1 ||
        blocks > 8 || (blocks & (blocks - 1)) != 0 || ((uintptr_t)q & 15) != 0 || q_stride % 8 != 0 ||
        ((uintptr_t)codes & 15) != 0 || ((uintptr_t)scales & 7) != 0 || ((uintptr_t)out & 7) != 0 ||
        (long long)pages * 2 * nkv * page_size > 0xffffffffll || (hd != 64 && hd != 128 && hd != 256))
        return -1;
    const Kv8DecodeArgs a{(const bf16*)q, (bf16*)out, (const uint8_t*)codes, (const uint8_t*)scales, block_table,
                          token_req, cache_pos, q_stride, bt_stride, bt_width, pages, nq, nkv, window, keep_first,
                          (nq / nkv + 7) / 8, scale * 1.4426950408889634f, page_split(page_size)};
    const cudaStream_t s = (cudaStream_t)stream;
    const bool few = nq / nkv <= 4;
    switch (hd) {
        case 64: return few ? launch_decode<64, 4>(a, tokens, blocks, warps, s) : launch_decode<64, 8>(a, tokens, blocks, warps, s);
        case 128: return few ? launch_decode<128, 4>(a, tokens, blocks, warps, s) : launch_decode<128, 8>(a, tokens, blocks, warps, s);
        default: return few ? launch_decode<256, 4>(a, tokens, blocks, warps, s) : launch_decode<256, 8>(a, tokens, blocks, warps, s);
    }
}

MSTAR_API int mstar_kv8_decode_packed(const long long* a) {
    return mstar_kv8_decode((const void*)a[0], (int)a[1], (void*)a[2], (const void*)a[3], (const void*)a[4],
        (int)a[5], (const int*)a[6], (int)a[7], (int)a[8], (const int*)a[9], (const int*)a[10], (int)a[11], (int)a[12],
        (int)a[13], (int)a[14], (int)a[15], (int)a[16], (int)a[17], kv8_packed_float(a[18]), (int)a[19], (int)a[20],
        (void*)a[21]);
}
