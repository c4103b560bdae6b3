// Grouped-query attention over the 8-bit cache (format: kv8.cuh) for the 32-bit mode and for what the other kernels do not
// take: prompt portions and single tokens, both activation types, any group of query heads, any page size.  Two kernels:
// head sizes 64, 128 and 256 on the tensor cores (second half of this file), others that are multiples of 8 up to 256 in
// float arithmetic on CUDA cores.
//
// On CUDA cores: a row is (token, query head of the group); R rows of one request and kv head make a block, which walks the
// keys that some of its rows see (kept first keys, then the window) in tiles of 64: codes become floats times their row's
// scale in shared memory (keys transposed), S = Q K^T and O += P V by outer products in registers, softmax statistics
// per row in registers.  R = 64 for portions (4 x 4 scores a thread), 8 for single tokens (a warp a row).  Where there
// are few row tiles the keys are cut into `splits` parts whose (maximum, sum, output) go to scratch memory.
//
// Semantics are those of attention_generic.cu; a row that sees no key gives zeros.
#include <cuda_fp16.h>

#include "kv8_merge.cuh"
#include "mma_util.cuh"

struct Kv8AttnArgs {
    const void* q;
    void* out;
    const uint8_t *codes, *scales;
    const int *block_table;
    // portions: first token and end of every entry, keys of every entry; single tokens: request and place of each
    const int *qo_indptr, *kv_len, *token_req, *cache_pos;
    int q_stride, bt_stride, bt_width, pages, nq, nkv, hd, window, keep_first, first_entry;
    float scale;
    PageSplit page;
    Kv8Parts parts;
};

template <typename A, int R>
__global__ void __launch_bounds__(256) kv8_attention_kernel(Kv8AttnArgs a) {
    constexpr int TX = R == 64 ? 16 : 32, RT = R * TX / 256, KT = 64 / TX, RP = R + 4, KP = 68, DT = 256 / TX;
    extern __shared__ __align__(16) float smem[];
    pdl_wait();
    const int hd = a.hd, G = a.nq / a.nkv;
    float* q_s = smem;                                   // [hd][RP]
    float* kv_s = q_s + hd * RP;                         // keys [hd][KP], then values [64][hd]
    float* p_s = kv_s + hd * KP;                         // [64][RP]
    __shared__ int bad_s[64];                            // keys whose key or value is NaNs
    const int tid = threadIdx.x, tx = tid % TX, ty = tid / TX;
    const int kvh = blockIdx.x / a.parts.splits, split = blockIdx.x % a.parts.splits;

    // the rows of this block: flattened (token, head of the group) from `row0` on
    int first_token, q_len, past, table_row;
    if (a.token_req != nullptr) {
        first_token = blockIdx.z;
        q_len = 1;
        past = a.cache_pos[first_token];
        table_row = a.token_req[first_token];
    } else {
        table_row = a.first_entry + blockIdx.z;
        first_token = a.qo_indptr[table_row];
        q_len = a.qo_indptr[table_row + 1] - first_token;
        past = a.kv_len[table_row] - q_len;
    }
    const int row0 = blockIdx.y * R, rows = q_len * G;
    if (row0 >= rows) return;
    const int last_row = min(row0 + R, rows) - 1;
    const int* bt = a.block_table + (size_t)table_row * a.bt_stride;
    SeenKeys seen = seen_keys(past + row0 / G, past + last_row / G, a.window, a.keep_first);
    const int part = a.parts.splits == 1 ? seen.count : ((seen.count + a.parts.splits - 1) / a.parts.splits + 63) & ~63;
    const int v_end = min(seen.count, (split + 1) * part);

    const A* q = (const A*)a.q;
    for (int i = tid; i < R * hd; i += 256) {
        const int r = i / hd, d = i - r * hd, row = row0 + r;
        float v = 0.f;
        if (row < rows) v = to_float(q[(size_t)(first_token + row / G) * a.q_stride + (size_t)(kvh * G + row % G) * hd + d]);
        q_s[d * RP + r] = v * a.scale;
    }
    int pos[RT];
    float m[RT], l[RT], acc[RT][DT];
#pragma unroll
    for (int r = 0; r < RT; ++r) {
        pos[r] = past + min(row0 + ty * RT + r, last_row) / G;
        m[r] = -INFINITY;
        l[r] = 0.f;
#pragma unroll
        for (int c = 0; c < DT; ++c) acc[r][c] = 0.f;
    }
    const int chunks = hd >> 3;
    const size_t plane = (size_t)a.nkv * a.page.size;

    for (int v0 = split * part; v0 < v_end; v0 += 64) {
        const int n = min(64, v_end - v0);
        float s[RT][KT];
#pragma unroll 1
        for (int which = 0; which < 2; ++which) {
            __syncthreads();
            // a tile of keys (transposed) or of values: 8 codes a thread and turn, the threads of a warp on different
            // rows.  Rows past the end are zeros.
            for (int i = tid; i < 64 * chunks; i += 256) {
                const int j = i & 63, d = (i >> 6) * 8;
                float v[8];
#pragma unroll
                for (int k = 0; k < 8; ++k) v[k] = 0.f;
                if (j < n) {
                    const int key = key_of(seen, v0 + j), logical = page_of(a.page, key);
                    const size_t at = ((size_t)page_id(bt, logical, a.bt_width, a.pages) * 2 + which) * plane +
                                      (size_t)kvh * a.page.size + (key - logical * a.page.size);
                    const uint2 w = *reinterpret_cast<const uint2*>(a.codes + at * hd + d);
                    const int byte = a.scales[at];
                    const float f = byte == KV8_BAD_BYTE ? 0.f : kv8_scale(byte);
                    if (which == 0 && d == 0) bad_s[j] = byte == KV8_BAD_BYTE || a.scales[at + plane] == KV8_BAD_BYTE;
                    kv8_unpack4(w.x, v);
                    kv8_unpack4(w.y, v + 4);
#pragma unroll
                    for (int k = 0; k < 8; ++k) v[k] *= f;
                }
                if (which == 0) {
#pragma unroll
                    for (int k = 0; k < 8; ++k) kv_s[(d + k) * KP + j] = v[k];
                } else {
                    store8(kv_s + j * hd + d, v);
                }
            }
            __syncthreads();
            if (which == 0) {
#pragma unroll
                for (int r = 0; r < RT; ++r)
#pragma unroll
                    for (int k = 0; k < KT; ++k) s[r][k] = 0.f;
#pragma unroll 4
                for (int d = 0; d < hd; ++d) {
                    float kd[KT];
                    if constexpr (KT == 4) {
                        const float4 k4 = *reinterpret_cast<const float4*>(kv_s + d * KP + tx * 4);
                        kd[0] = k4.x; kd[1] = k4.y; kd[2] = k4.z; kd[3] = k4.w;
                        const float4 q4 = *reinterpret_cast<const float4*>(q_s + d * RP + ty * 4);
                        const float qd[4] = {q4.x, q4.y, q4.z, q4.w};
#pragma unroll
                        for (int r = 0; r < RT; ++r)
#pragma unroll
                            for (int k = 0; k < KT; ++k) s[r][k] = fmaf(qd[r], kd[k], s[r][k]);
                    } else {
                        const float2 k2 = *reinterpret_cast<const float2*>(kv_s + d * KP + tx * 2);
                        const float qd = q_s[d * RP + ty];
                        s[0][0] = fmaf(qd, k2.x, s[0][0]);
                        s[0][1] = fmaf(qd, k2.y, s[0][1]);
                    }
                }
                // the running softmax; rows of a half warp (R = 64) or of a warp
#pragma unroll
                for (int r = 0; r < RT; ++r) {
                    float mx = -INFINITY;
#pragma unroll
                    for (int k = 0; k < KT; ++k) {
                        const int v = tx * KT + k;
                        if (v >= n || !sees(pos[r], key_of(seen, v0 + v), a.window, a.keep_first)) s[r][k] = -INFINITY;
                        else if (bad_s[v]) s[r][k] = __int_as_float(0x7fc00000);
                        mx = fmaxf(mx, s[r][k]);
                    }
#pragma unroll
                    for (int o = TX / 2; o > 0; o >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, o));
                    const float now = fmaxf(m[r], mx);
                    // nothing seen so far: the weights below are exp(-inf) = 0 whatever finite number is taken off
                    const float ref = now == -INFINITY ? 0.f : now;
                    const float alpha = expf(m[r] - ref);
                    float sum = 0.f;
#pragma unroll
                    for (int k = 0; k < KT; ++k) {
                        s[r][k] = expf(s[r][k] - ref);
                        sum += s[r][k];
                    }
#pragma unroll
                    for (int o = TX / 2; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
                    m[r] = now;
                    l[r] = l[r] * alpha + sum;
#pragma unroll
                    for (int c = 0; c < DT; ++c) acc[r][c] *= alpha;
                }
                // the whole row of weights, so that the values' product needs no other thread's registers
#pragma unroll
                for (int k = 0; k < KT; ++k)
#pragma unroll
                    for (int r = 0; r < RT; ++r) p_s[(tx * KT + k) * RP + ty * RT + r] = s[r][k];
            } else {
                for (int j = 0; j < n; ++j) {
                    float p[RT];
#pragma unroll
                    for (int r = 0; r < RT; ++r) p[r] = p_s[j * RP + ty * RT + r];
#pragma unroll
                    for (int c = 0; c < DT; ++c) {
                        const int d = tx + c * TX;
                        if (d < hd) {
                            const float v = kv_s[j * hd + d];
#pragma unroll
                            for (int r = 0; r < RT; ++r) acc[r][c] = fmaf(p[r], v, acc[r][c]);
                        }
                    }
                }
            }
        }
    }
    pdl_launch_dependents();
#pragma unroll
    for (int r = 0; r < RT; ++r) {
        const int row = row0 + ty * RT + r;
        if (row >= rows) continue;
        const size_t head = (size_t)(first_token + row / G) * a.nq + kvh * G + row % G;
        if (a.parts.splits == 1) {
            const float inv = l[r] == 0.f ? 0.f : 1.f / l[r];
#pragma unroll
            for (int c = 0; c < DT; ++c)
                if (tx + c * TX < hd) ((A*)a.out)[head * hd + tx + c * TX] = from_float<A>(acc[r][c] * inv);
        } else if (kv8_has_room(a.parts, first_token + row / G)) {
            const size_t at = (head - (size_t)kv8_first_token(a.parts) * a.nq) * a.parts.splits + split;
#pragma unroll
            for (int c = 0; c < DT; ++c)
                if (tx + c * TX < hd) a.parts.o[at * hd + tx + c * TX] = acc[r][c];
            if (tx == 0) {
                a.parts.ml[2 * at] = m[r] * 1.4426950408889634f;
                a.parts.ml[2 * at + 1] = l[r];
            }
        }
    }
}

template <typename A, int R> static int launch_simt(const Kv8AttnArgs& a, dim3 grid, cudaStream_t s) {
    const int smem = (a.hd * (R + 4) + a.hd * 68 + 64 * (R + 4)) * (int)sizeof(float);
    auto kernel = kv8_attention_kernel<A, R>;
    static bool configured[64] = {false};
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return (int)e;
    if (dev < 0 || dev >= 64) return -1;
    if (!configured[dev]) {
        e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, 224 * 1024);
        if (e != cudaSuccess) return (int)e;
        configured[dev] = true;
    }
    e = mstar_launch(kernel, grid, dim3(256), (size_t)smem, s, a);
    return e != cudaSuccess ? (int)e : launch_status();
}

// ---------------------------------------------------------------------------------------- on the tensor cores
// Scores: m16n8k16 products of float16 with float sums.  e4m3 is exact in float16, so the codes of keys are converted in
// registers; a row of queries is scaled by a power of two to have its largest number in [2^13, 2^14) and is one float16
// (exact for a bfloat16 but for numbers 2^-27 below the largest), in the 32-bit mode two, x = hi + lo: within 2^-22 of a number
// or 2^-38 of the row's largest, a product each.  The keys' scales are factors of the scores.
//
// Outputs: products of bfloat16.  Values become bfloat16 with their row's scale, which is exact for every scale (kv8.cuh), and
// weights 2^(s_j - m) are two bfloat16 parts in the 16-bit mode (16 bits), three in the 32-bit mode (all 24 bits of a float),
// down to 2^-126 of the largest: a small weight, or a row of small values beside one of large values, keeps its bits.
// (Weights in float16 relative to the largest 2^(s_j + e_j), with the values' exponents in them, took a product less, but what
// lay 2^25 below the largest was lost in every feature.  Times so: 15.8, 327, 103, 18.4 us for the four calls below.)
//
// The tensor cores cut the sums that they add to instead of rounding them: over 6,500 keys that was 1.2e-5 of the output, all
// one way.  So in the 32-bit mode a tile's products are summed from zero and added in float arithmetic (9.5e-7; 359 us for
// the two portions of 512 tokens below instead of 350), over 4 or 8 blocks of 8 features at a time, as the registers allow
// (4 of heads of 64: 435 us; 8 of heads of 256, 100 tokens on 2,000: 79.5 instead of 72.9; 8 with few rows: 24.3, not 23.4).
//
// A warp owns 16 rows (token, query head of the group) and, of every tile of 64 keys, 8 NT: with NT 8 a block's four
// warps have 64 rows, with NT 2 (16 rows or fewer) they share a tile's keys and leave a part each.  Tiles of codes come by
// cp.async, one tile ahead (three with few rows), into swizzled shared memory.  Which features and keys the elements of the
// scores' operands are is chosen as in the decode kernel, and the queries lie in shared memory in that order.  The values of a
// tile are converted once, each warp a quarter of the keys (with NT 2 its own), into a bfloat16 tile.
//
// Bound by instructions and the tensor pipe.  In the 32-bit mode two portions of 251 tokens, 32 heads of 64 over 8, a window of
// 200, take 15.8 us (on CUDA cores 108), two of 512 on 6,000 cached 359 (112 TFLOP/s; five products for two), in the 16-bit
// mode 512 tokens of 12 heads of 256 over 4 on 2,000 cached 141; float single tokens of 8 requests on 800 to 2,048 keys, 24
// heads of 128 over 8, 23 us.
__device__ __forceinline__ uint32_t f16x2_of_codes(uint32_t two) {
    uint32_t r;
    asm("{\n\t.reg .b16 lo, hi;\n\tmov.b32 {lo, hi}, %1;\n\tcvt.rn.f16x2.e4m3x2 %0, lo;\n\t}" : "=r"(r) : "r"(two));
    return r;
}
__device__ __forceinline__ uint32_t f16x2_of_codes_hi(uint32_t two) {
    uint32_t r;
    asm("{\n\t.reg .b16 lo, hi;\n\tmov.b32 {lo, hi}, %1;\n\tcvt.rn.f16x2.e4m3x2 %0, hi;\n\t}" : "=r"(r) : "r"(two));
    return r;
}
__device__ __forceinline__ void mma_f16_16816(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};\n"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ float exp2_approx(float x) {
    float y;
    asm("ex2.approx.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ uint32_t f16x2(float lo, float hi) {
    const __half2 v = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&v);
}
__device__ __forceinline__ float2 floats_of(uint32_t two) { return __half22float2(*reinterpret_cast<const __half2*>(&two)); }
// Two neighbouring elements
__device__ __forceinline__ void store2(float* p, float a, float b) { *reinterpret_cast<float2*>(p) = make_float2(a, b); }
__device__ __forceinline__ void store2(bf16* p, float a, float b) { *reinterpret_cast<uint32_t*>(p) = pack_bf16(a, b); }

#define KM_SLACK 8.f
template <int HD> __host__ __device__ constexpr int km_tile() { return 64 * HD; }
// tiles of which a block holds copies, on the way or there: with few rows a tile is soon worked off
template <int NT> __host__ __device__ constexpr int km_stages() { return NT == 8 ? 2 : 4; }
template <int HD, int PARTS, int NT> __host__ __device__ constexpr int km_smem() {
    return km_stages<NT>() * (2 * km_tile<HD>() + 64 * 12) + 2 * km_tile<HD>() + PARTS * (NT == 8 ? 64 : 16) * (HD * 2 + 16) + 64 * 4;
}

template <typename A, int HD, int PARTS, int NT>
__global__ void __launch_bounds__(128) kv8_attention_mma_kernel(Kv8AttnArgs a) {
    constexpr int ROWS = NT == 8 ? 64 : 16, RB = HD < 128 ? HD : 128, KC = HD / 64, MT = HD / 8;
    constexpr int PP = PARTS + 1;                        // parts of a weight
    constexpr int KB = NT == 8 && HD < 256 ? 8 : 4;      // blocks of 8 features that are summed side by side
    constexpr int NB = NT < 4 ? NT : 4;                  // products side by side
    constexpr int QP = HD * 2 + 16;                      // bytes of a row of queries in shared memory
    constexpr int S = km_stages<NT>();
    extern __shared__ __align__(128) unsigned char smem_m[];
    unsigned char* k_s = smem_m;                         // [S][64 keys x HD codes], then values
    unsigned char* v_s = k_s + S * km_tile<HD>();
    unsigned char* b_s = v_s + S * km_tile<HD>();        // [64 keys x HD bfloat16]: a tile's values
    unsigned char* q_s = b_s + 2 * km_tile<HD>();        // [PARTS][ROWS][QP]
    // [S][64] 2^e of the key, the value's factors as bits
    float2* sc_s = reinterpret_cast<float2*>(q_s + PARTS * ROWS * QP);
    uint32_t* row_s = reinterpret_cast<uint32_t*>(sc_s + S * 64);         // [S][64]
    float* qscale_s = reinterpret_cast<float*>(row_s + S * 64);           // [ROWS]
    pdl_wait();
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t = lane & 3, G = a.nq / a.nkv;
    const int ranges = NT == 8 ? a.parts.splits : max(1, a.parts.splits / 4);      // ranges of keys; a part a warp, or one
    const int kvh = blockIdx.x / ranges, range = blockIdx.x % ranges;
    int first_token, q_len, past, table_row;
    if (a.token_req != nullptr) {
        first_token = blockIdx.z;
        q_len = 1;
        past = a.cache_pos[first_token];
        table_row = a.token_req[first_token];
    } else {
        table_row = a.first_entry + blockIdx.z;
        first_token = a.qo_indptr[table_row];
        q_len = a.qo_indptr[table_row + 1] - first_token;
        past = a.kv_len[table_row] - q_len;
    }
    const int row0 = blockIdx.y * ROWS, rows = q_len * G;
    if (row0 >= rows) return;
    const int last_row = min(row0 + ROWS, rows) - 1;
    const int* bt = a.block_table + (size_t)table_row * a.bt_stride;
    const SeenKeys seen = seen_keys(past + row0 / G, past + last_row / G, a.window, a.keep_first);
    const int all = (seen.count + 63) >> 6, per = (all + ranges - 1) / ranges;
    const int tile0 = range * per, tiles = max(0, min(per, all - tile0));
    const size_t plane = (size_t)a.nkv * a.page.size;

    // ---- queries: LR lanes a row, four features a lane and load, NQ loads a turn.  The first turn's go before all else.
    constexpr int LR = HD < 128 ? HD / 4 : 32, NL = HD / 4 / LR, NQ = NT == 8 ? 8 : 4 * NL * LR / 32;
    constexpr int RT = NQ / NL * (32 / LR), TURNS = ROWS / 4 / RT;           // rows of a turn of a warp
    const bool wide = a.q_stride % 4 == 0 && ((uintptr_t)a.q & 15) == 0;
    float qv[NQ][4];
    auto q_row = [&](int turn, int i) { return warp * (ROWS / 4) + turn * RT + i / NL * (32 / LR) + lane / LR; };
    auto q_feature = [&](int i) { return i % NL * 128 + lane % LR * 4; };
    auto load_q = [&](int turn) {
#pragma unroll
        for (int i = 0; i < NQ; ++i) {
            const int row = row0 + q_row(turn, i);
            const A* q = (const A*)a.q + (size_t)(first_token + min(row, last_row) / G) * a.q_stride +
                         (size_t)(kvh * G + min(row, last_row) % G) * HD + q_feature(i);
            if (wide) {
                load4(q, qv[i]);
            } else {
#pragma unroll
                for (int j = 0; j < 4; ++j) qv[i][j] = to_float(q[j]);
            }
        }
    };
    // row r's feature d at the place that the fragments want: of 64 features, 16 t + 4 s + e is k-step s, element
    // 2 t + e % 2 + 8 (e / 2)
    auto keep_q = [&](int turn) {
#pragma unroll
        for (int i0 = 0; i0 < NQ; i0 += NL) {
            float most = 0.f;
#pragma unroll
            for (int i = i0; i < i0 + NL; ++i)
#pragma unroll
                for (int j = 0; j < 4; ++j) most = fabsf(qv[i][j]) < INFINITY ? fmaxf(most, fabsf(qv[i][j])) : INFINITY;
#pragma unroll
            for (int o = LR / 2; o > 0; o >>= 1) most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, o));
            // (one below 2^-113 is taken as that large, so that the factors are normal numbers)
            const uint32_t e = max(__float_as_uint(most) >> 23, 14u);
            const float down = e < 255u ? __uint_as_float((267u - e) << 23) : 0.f;
            const int r = q_row(turn, i0);
            if (lane % LR == 0)
                qscale_s[r] = e < 255u ? __uint_as_float((e - 13u) << 23) * a.scale * 1.4426950408889634f : __int_as_float(0x7fc00000);
#pragma unroll
            for (int i = i0; i < i0 + NL; ++i) {
                const int d = q_feature(i), x = d & 63;
                unsigned char* to = q_s + r * QP + ((d & ~63) + ((x >> 2) & 3) * 16 + 2 * (x >> 4)) * 2;
#pragma unroll
                for (int j = 0; j < 2; ++j) {
                    const float y0 = e < 255u ? qv[i][2 * j] * down : 0.f, y1 = e < 255u ? qv[i][2 * j + 1] * down : 0.f;
                    const uint32_t hi = f16x2(y0, y1);
                    *reinterpret_cast<uint32_t*>(to + 16 * j) = hi;
                    if constexpr (PARTS == 2) {
                        const float2 b = floats_of(hi);
                        *reinterpret_cast<uint32_t*>(to + ROWS * QP + 16 * j) = f16x2(y0 - b.x, y1 - b.y);
                    }
                }
            }
        }
    };
    load_q(0);

    // ---- rows, scales and copies of tiles; the table's entries are read a tile ahead of the rows, the scales a tile
    // ahead of their use
    auto key_at = [&](int i) { return key_of(seen, min((tile0 + i) * 64 + tid, seen.count - 1)); };
    int entry[S], ks = 0, vs = 0;
    auto ask_entry = [&](int i, int& to) {
        if (tid < 64 && i < tiles) to = bt[min(page_of(a.page, key_at(i)), a.bt_width - 1)];
    };
    auto keep_row = [&](int i, int from) {
        if (tid < 64 && i < tiles) {
            const int key = key_at(i), page = (int)min((unsigned)from, (unsigned)(a.pages - 1));
            const uint32_t row = ((uint32_t)page * 2 * a.nkv + kvh) * a.page.size + (uint32_t)(key - page_of(a.page, key) * a.page.size);
            row_s[i % S * 64 + tid] = row;
            ks = a.scales[row];
            vs = a.scales[row + plane];
        }
    };
    auto keep_scales = [&](int i) {
        if (tid < 64 && i < tiles) {
            const bool bad = ks == KV8_BAD_BYTE || vs == KV8_BAD_BYTE;
            sc_s[i % S * 64 + tid] = make_float2(bad ? __int_as_float(0x7fc00000) : kv8_scale(ks),
                                                     __uint_as_float(kv8_value_factors(bad ? 0 : vs - 127)));
        }
    };
    // where a 16-byte run c of row r lies in a block of a tile: the swizzle of 128- or 64-byte rows
    auto at = [](int r, int c) { return r * RB + ((RB == 128 ? c ^ (r & 7) : c ^ ((r >> 1) & 3)) << 4); };
    auto copy = [&](int i) {
        if (i < tiles) {
            constexpr int CPR = HD / 16;
#pragma unroll
            for (int k = 0; k < CPR / 2; ++k) {
                const int r = (k * 128 + tid) / CPR, run = tid % CPR;
                const uint8_t* src = a.codes + (size_t)row_s[i % S * 64 + r] * HD + run * 16;
                const uint32_t to = smem_u32(k_s) + i % S * km_tile<HD>() + (run >> 3) * (64 * RB) + at(r, run & 7);
                cp_async_16(to, src, 16);
                cp_async_16(to + S * km_tile<HD>(), src + plane * HD, 16);
            }
        }
        cp_async_commit();
    };
#pragma unroll
    for (int i = 0; i < S; ++i) ask_entry(i, entry[i]);
#pragma unroll
    for (int i = 0; i < S - 1; ++i) {
        if (i > 0) keep_scales(i - 1);
        keep_row(i, entry[i]);
    }
    entry[0] = entry[S - 1];
    __syncthreads();
#pragma unroll
    for (int i = 0; i < S - 1; ++i) copy(i);
#pragma unroll
    for (int i = 0; i < TURNS; ++i) {
        if (i > 0) load_q(i);
        keep_q(i);
    }
    __syncthreads();
    const int wr = NT == 8 ? warp * 16 : 0, n0 = NT == 8 ? 0 : warp * NT;      // the warp's rows, its first 8 keys of a tile
    const float qs[2] = {qscale_s[wr + g], qscale_s[wr + g + 8]};
    // which of the keys in sight (counted as in SeenKeys) a row sees: those up to `last`, of these from `first` on or
    // before `kept`.  A row sees all keys below a block's last `first` and above its first `last`.
    const int shift = seen.kept - seen.lo, kept = max(seen.kept, a.keep_first + shift);
    auto last_of = [&](int row) { return past + row / G + shift; };
    auto first_of = [&](int row) { return a.window > 0 ? last_of(row) - a.window + 1 : 0; };
    int last[2], first[2];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        last[h] = last_of(min(row0 + wr + g + 8 * h, last_row));
        first[h] = first_of(min(row0 + wr + g + 8 * h, last_row));
    }

    float o[MT][4], m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f};
#pragma unroll
    for (int i = 0; i < MT; ++i) o[i][0] = o[i][1] = o[i][2] = o[i][3] = 0.f;
    const int kg = (g & 1) ? g ^ 4 : g, kt = (2 * t + 1) ^ 4;      // a product's row or key i is key i, or i ^ 4 where i is odd
    // the row (key of 16) and the 16-byte run of features that this lane names of the values' four matrices of 8 x 8
    const int vr = (lane & 1 ? (lane & 7) ^ 4 : lane & 7) + (lane & 8), vc = lane >> 4;
    const uint32_t q_at = smem_u32(q_s) + (wr + (lane & 15)) * QP + (lane >> 4) * 16;

    for (int i = 0; i < tiles; ++i) {
        keep_scales(i + S - 2);
        keep_row(i + S - 1, entry[0]);
        ask_entry(i + S, entry[0]);
        cp_async_wait<S - 2>();
        __syncthreads();                                 // this tile is there, the next rows are, the last tile's place is free
        copy(i + S - 1);
        const unsigned char* kt_s = k_s + i % S * km_tile<HD>();
        const unsigned char* vt_s = v_s + i % S * km_tile<HD>();
        const float2* sc = sc_s + i % S * 64;
        const int v0 = (tile0 + i) * 64;
        // ---- values: a run of 16 codes a lane and turn, of the warp's 16 keys, becomes two runs of 16 bytes
        {
            constexpr int CPR = HD / 16, BR = HD * 2;
#pragma unroll
            for (int k = 0; k < CPR / 2; ++k) {
                const int r = warp * 16 + (k * 32 + lane) / CPR, run = lane % CPR;
                const uint4 x = *reinterpret_cast<const uint4*>(vt_s + (run >> 3) * (64 * RB) + at(r, run & 7));
                uint32_t y[8];
                kv8_values16(x, __float_as_uint(sc[r].y), y);
                // (the runs of a row that lie 128 bytes apart take their two stores in the other order: different banks)
                const int odd = (run >> 2) & 1;
                unsigned char* to = b_s + r * BR;
                *reinterpret_cast<uint4*>(to + (((2 * run + odd) ^ (r & 7)) << 4)) =
                    odd ? make_uint4(y[4], y[5], y[6], y[7]) : make_uint4(y[0], y[1], y[2], y[3]);
                *reinterpret_cast<uint4*>(to + (((2 * run + 1 - odd) ^ (r & 7)) << 4)) =
                    odd ? make_uint4(y[0], y[1], y[2], y[3]) : make_uint4(y[4], y[5], y[6], y[7]);
            }
        }
        // ---- scores: s[n][2h + k], row g + 8h, keys 8 (n0 + n) + 2t and + kt
        float s[NT][4];
#pragma unroll
        for (int n = 0; n < NT; ++n) s[n][0] = s[n][1] = s[n][2] = s[n][3] = 0.f;
#pragma unroll
        for (int c = 0; c < KC; ++c) {
            uint32_t qf[PARTS][4][4];
#pragma unroll
            for (int p = 0; p < PARTS; ++p)
#pragma unroll
                for (int k = 0; k < 4; ++k) ldmatrix_x4(qf[p][k], q_at + p * ROWS * QP + (c * 4 + k) * 32);
#pragma unroll
            for (int n = 0; n < NT; n += NB) {             // NB products side by side: one waits for the last into its sum
                uint32_t b[NB][4];
#pragma unroll
                for (int y = 0; y < NB; ++y) {
                    const uint4 x = *reinterpret_cast<const uint4*>(kt_s + (c >> 1) * (64 * RB) + at((n0 + n + y) * 8 + kg, t + 4 * (c & 1)));
                    b[y][0] = x.x; b[y][1] = x.y; b[y][2] = x.z; b[y][3] = x.w;
                }
#pragma unroll
                for (int k = 0; k < 4; ++k)
#pragma unroll
                    for (int p = 0; p < PARTS; ++p)
#pragma unroll
                        for (int y = 0; y < NB; ++y)
                            mma_f16_16816(s[n + y], qf[p][k], f16x2_of_codes(b[y][k]), f16x2_of_codes_hi(b[y][k]));
            }
        }
        // ---- weights
        float top[2] = {-INFINITY, -INFINITY};
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int k = 0; k < 2; ++k) {
                const float f = sc[(n0 + n) * 8 + (k ? kt : 2 * t)].x;
#pragma unroll
                for (int h = 0; h < 2; ++h) s[n][2 * h + k] *= f * qs[h];
            }
        if (v0 + 63 > last_of(row0) || (v0 < first_of(last_row) && v0 + 63 >= kept)) {
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
                for (int k = 0; k < 2; ++k) {
                    const int v = v0 + (n0 + n) * 8 + (k ? kt : 2 * t);
#pragma unroll
                    for (int h = 0; h < 2; ++h)
                        if (v > last[h] || (v < first[h] && v >= kept)) s[n][2 * h + k] = -INFINITY;
                }
        }
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int j = 0; j < 4; ++j) top[j >> 1] = fmaxf(top[j >> 1], s[n][j]);
        // m: what scores are taken off from, at least the largest so far and 2^KM_SLACK above it where it was set, so that no
        // weight is above 1 and the sums of values no larger than values are
        if (__any_sync(0xffffffffu, (top[0] > m[0]) | (top[1] > m[1]))) {
            float up[2];
#pragma unroll
            for (int h = 0; h < 2; ++h) {
#pragma unroll
                for (int d = 1; d < 4; d <<= 1) top[h] = fmaxf(top[h], __shfl_xor_sync(0xffffffffu, top[h], d));
                const float now = top[h] > m[h] ? top[h] + KM_SLACK : m[h];
                up[h] = m[h] == -INFINITY ? 1.f : exp2_approx(m[h] - now);      // (l is 0 or NaN, o zeros or NaNs, where it is -inf)
                l[h] *= up[h];
                m[h] = now;
            }
#pragma unroll
            for (int k = 0; k < MT; ++k) {
                o[k][0] *= up[0];
                o[k][1] *= up[0];
                o[k][2] *= up[1];
                o[k][3] *= up[1];
            }
        }
        const float mr[2] = {m[0] == -INFINITY ? 0.f : m[0], m[1] == -INFINITY ? 0.f : m[1]};
        // the values are there: of all warps, or of this one
        if constexpr (NT == 8) __syncthreads();
        else __syncwarp();
        // ---- outputs.  In the 32-bit mode the tile's products are summed by themselves and then added, which rounds
        uint32_t pf[NT / 2][PP][4];
#pragma unroll
        for (int u = 0; u < NT / 2; ++u)
#pragma unroll
            for (int x = 0; x < 2; ++x)
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    const int n = 2 * u + x;
                    float p0 = exp2_approx(s[n][2 * h] - mr[h]), p1 = exp2_approx(s[n][2 * h + 1] - mr[h]);
                    l[h] += p0 + p1;
#pragma unroll
                    for (int p = 0; p < PP; ++p) {       // what the parts before leave, rounded
                        const uint32_t b = pack_bf16(p0, p1);
                        pf[u][p][2 * x + h] = b;
                        p0 -= __uint_as_float(b << 16);
                        p1 -= __uint_as_float(b & 0xffff0000u);
                    }
                }
#pragma unroll
        for (int k = 0; k < MT; k += KB) {               // KB blocks of 8 features
            float sum[KB][4];
#pragma unroll
            for (int i = 0; i < KB; ++i)
#pragma unroll
                for (int e = 0; e < 4; ++e) sum[i][e] = PARTS == 2 ? 0.f : o[k + i][e];
#pragma unroll
            for (int u = 0; u < NT / 2; ++u) {
                const int r = (n0 + 2 * u) * 8 + vr;
                uint32_t v[KB / 2][4];
#pragma unroll
                for (int i = 0; i < KB / 2; ++i)
                    ldmatrix_x4_trans(v[i], smem_u32(b_s) + r * (HD * 2) + (((k + 2 * i + vc) ^ (r & 7)) << 4));
#pragma unroll
                for (int p = PP - 1; p >= 0; --p)        // (the small parts first)
#pragma unroll
                    for (int i = 0; i < KB; ++i) mma_bf16_16816(sum[i], pf[u][p], v[i / 2][2 * (i & 1)], v[i / 2][2 * (i & 1) + 1]);
            }
#pragma unroll
            for (int i = 0; i < KB; ++i)
#pragma unroll
                for (int e = 0; e < 4; ++e) o[k + i][e] = PARTS == 2 ? o[k + i][e] + sum[i][e] : sum[i][e];
        }
    }
    cp_async_wait<0>();
    pdl_launch_dependents();
    // ---- the rows' sums, and the outputs: o[k][2h + e], row g + 8h, feature 8 k + 2 t + e
    const int part = NT == 8 ? range : range * 4 + warp;
    const bool parts = NT == 2 || a.parts.splits > 1;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
#pragma unroll
        for (int d = 1; d < 4; d <<= 1) l[h] += __shfl_xor_sync(0xffffffffu, l[h], d);
        const int row = row0 + wr + g + 8 * h;
        if (row >= rows || (parts && !kv8_has_room(a.parts, first_token + row / G))) continue;
        const size_t head = (size_t)(first_token + row / G) * a.nq + kvh * G + row % G;
        const size_t at_part = (head - (size_t)kv8_first_token(a.parts) * a.nq) * a.parts.splits + part;
        if (parts && t == 0) {
            a.parts.ml[2 * at_part] = m[h];
            a.parts.ml[2 * at_part + 1] = l[h];
        }
        const float f = parts ? 1.f : l[h] == 0.f ? 0.f : 1.f / l[h];
#pragma unroll
        for (int k = 0; k < MT; ++k) {
            const int d = 8 * k + 2 * t;
            if (parts) store2(a.parts.o + at_part * HD + d, o[k][2 * h], o[k][2 * h + 1]);
            else store2((A*)a.out + head * HD + d, o[k][2 * h] * f, o[k][2 * h + 1] * f);
        }
    }
}

template <typename A, int HD, int PARTS, int NT>
static int launch_mma(const Kv8AttnArgs& a, dim3 grid, cudaStream_t s) {
    auto kernel = kv8_attention_mma_kernel<A, HD, PARTS, NT>;
    constexpr int smem = km_smem<HD, PARTS, NT>();
    static bool configured[64] = {false};
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return (int)e;
    if (dev < 0 || dev >= 64) return -1;
    if (!configured[dev]) {
        e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
        if (e != cudaSuccess) return (int)e;
        configured[dev] = true;
    }
    e = mstar_launch(kernel, grid, dim3(128), (size_t)smem, s, a);
    return e != cudaSuccess ? (int)e : launch_status();
}
template <typename A, int PARTS, int NT> static int launch_mma_hd(const Kv8AttnArgs& a, dim3 grid, cudaStream_t s) {
    switch (a.hd) {
        case 64: return launch_mma<A, 64, PARTS, NT>(a, grid, s);
        case 128: return launch_mma<A, 128, PARTS, NT>(a, grid, s);
        default: return launch_mma<A, 256, PARTS, NT>(a, grid, s);
    }
}

// Portions (token_req null): entries [first_entry, first_entry + count) of at most max_q tokens.  Single tokens:
// tokens [0, count).  `tokens`: at least as many as the call covers, at most what `out` has.  splits > 1: the keys of a
// row tile are cut into that many parts, `part_o` (tokens * nq * splits * hd floats) and `part_ml` (2 each) hold their
// parts and a second kernel joins them; a multiple of 4 where rows are 16 or fewer and hd is 64, 128 or 256 (a part a
// warp).  Returns 0, a CUDA error code or -1 (shape refused).
MSTAR_API int mstar_kv8_attention(const void* q, int q_stride, void* out, int act_dtype, const void* codes,
                                  const void* scales, int pages, const int* block_table, int bt_stride, int bt_width,
                                  const int* qo_indptr, const int* kv_len, const int* token_req, const int* cache_pos,
                                  int first_entry, int count, int max_q, int tokens, int nq, int nkv, int hd,
                                  int page_size, int window, int keep_first, float scale, int splits, float* part_o,
                                  float* part_ml, void* stream) {
    if (count <= 0 || max_q <= 0) return 0;
    if (hd <= 0 || hd % 8 != 0 || hd > 256 || nkv <= 0 || nq % nkv != 0 || page_size <= 0 || pages <= 0 || bt_width <= 0 ||
        splits < 1 || count > 65535 || ((uintptr_t)codes & 7) != 0 || ((uintptr_t)out & 15) != 0)
        return -1;
    const Kv8Parts parts{part_o, part_ml, splits, token_req == nullptr ? qo_indptr + first_entry : nullptr, count, tokens};
    const Kv8AttnArgs a{q, out, (const uint8_t*)codes, (const uint8_t*)scales, block_table, qo_indptr, kv_len, token_req,
                        cache_pos, q_stride, bt_stride, bt_width, pages, nq, nkv, hd, window, keep_first, first_entry, scale,
                        page_split(page_size), parts};
    const long long rows = (long long)max_q * (nq / nkv);
    const cudaStream_t s = (cudaStream_t)stream;
    int code;
    // (the copies want runs of 16 bytes)
    if ((hd == 64 || hd == 128 || hd == 256) && ((uintptr_t)codes & 15) == 0 &&
        (long long)pages * 2 * nkv * page_size <= 0xffffffffll) {
        const bool few = rows <= 16;
        if (few && splits % 4 != 0) return -1;
        const long long tiles = few ? 1 : (rows + 63) / 64;
        if (tiles > 65535) return -1;
        const dim3 grid(nkv * (few ? splits / 4 : splits), (unsigned)tiles, count);
        if (act_dtype == MSTAR_F32) code = few ? launch_mma_hd<float, 2, 2>(a, grid, s) : launch_mma_hd<float, 2, 8>(a, grid, s);
        else code = few ? launch_mma_hd<bf16, 1, 2>(a, grid, s) : launch_mma_hd<bf16, 1, 8>(a, grid, s);
    } else {
        const int R = rows <= 8 ? 8 : 64;
        const long long tiles = (rows + R - 1) / R;
        if (tiles > 65535) return -1;
        const dim3 grid(nkv * splits, (unsigned)tiles, count);
        if (act_dtype == MSTAR_F32) code = R == 8 ? launch_simt<float, 8>(a, grid, s) : launch_simt<float, 64>(a, grid, s);
        else code = R == 8 ? launch_simt<bf16, 8>(a, grid, s) : launch_simt<bf16, 64>(a, grid, s);
    }
    if (code != 0 || splits == 1) return code;
    return kv8_merge(parts, out, act_dtype, nq, hd, s);
}

MSTAR_API int mstar_kv8_attention_packed(const long long* a) {
    return mstar_kv8_attention((const void*)a[0], (int)a[1], (void*)a[2], (int)a[3], (const void*)a[4],
        (const void*)a[5], (int)a[6], (const int*)a[7], (int)a[8], (int)a[9], (const int*)a[10], (const int*)a[11],
        (const int*)a[12], (const int*)a[13], (int)a[14], (int)a[15], (int)a[16], (int)a[17], (int)a[18], (int)a[19],
        (int)a[20], (int)a[21], (int)a[22], (int)a[23], kv8_packed_float(a[24]), (int)a[25], (float*)a[26],
        (float*)a[27], (void*)a[28]);
}
