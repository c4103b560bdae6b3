// Grouped-query attention over the 8-bit cache (format: kv8.cuh) in float arithmetic on CUDA cores: prompt portions
// and single tokens, both activation types, any head size that is a multiple of 8 up to 256, any group of query
// heads, any page size.  It is the attention of the 32-bit mode and of the shapes that the tensor-core kernels do not
// take.
//
// A row is (token, query head of the group); R rows of one request and kv head make a block, which walks the keys
// that some of its rows see (kept first keys, then the window) in tiles of 64: codes become floats times their row's
// scale in shared memory (keys transposed), S = Q K^T and O += P V by outer products in registers, softmax statistics
// per row in registers.  R = 64 for portions (4 x 4 scores a thread), 8 for single tokens (a warp a row).  Where there
// are few row tiles the keys are cut into `splits` parts whose (maximum, sum, output) go to scratch memory.
//
// Semantics are those of attention_generic.cu; a row that sees no key gives zeros.
#include "kv8_merge.cuh"

struct Kv8AttnArgs {
    const void* q;
    void* out;
    const uint8_t *codes, *scales;
    const int *block_table;
    // portions: first token and end of every entry, keys of every entry; single tokens: request and place of each
    const int *qo_indptr, *kv_len, *token_req, *cache_pos;
    int q_stride, bt_stride, pages, nq, nkv, hd, window, keep_first, first_entry;
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
                    const size_t at = ((size_t)page_id(bt, logical, a.bt_stride, a.pages) * 2 + which) * plane +
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
        } else {
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
    static int configured = 0;
    if (smem > configured) {
        const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, 224 * 1024);
        if (e != cudaSuccess) return (int)e;
        configured = 224 * 1024;
    }
    const cudaError_t e = mstar_launch(kernel, grid, dim3(256), (size_t)smem, s, a);
    return e != cudaSuccess ? (int)e : launch_status();
}

// Portions (token_req null): entries [first_entry, first_entry + count) of at most max_q tokens.  Single tokens:
// tokens [0, count).  `tokens`: at least as many as the call covers, at most what `out` has.  splits > 1: the keys of a
// row tile are shared by that many blocks, `part_o` (tokens * nq * splits * hd floats) and `part_ml` (2 each) hold their
// parts and a second kernel joins them.  Returns 0, a CUDA error code or -1 (shape refused).
MSTAR_API int mstar_kv8_attention(const void* q, int q_stride, void* out, int act_dtype, const void* codes,
                                  const void* scales, int pages, const int* block_table, int bt_stride,
                                  const int* qo_indptr, const int* kv_len, const int* token_req, const int* cache_pos,
                                  int first_entry, int count, int max_q, int tokens, int nq, int nkv, int hd,
                                  int page_size, int window, int keep_first, float scale, int splits, float* part_o,
                                  float* part_ml, void* stream) {
    if (count <= 0 || max_q <= 0) return 0;
    if (hd <= 0 || hd % 8 != 0 || hd > 256 || nkv <= 0 || nq % nkv != 0 || page_size <= 0 || pages <= 0 || splits < 1 ||
        count > 65535 || ((uintptr_t)codes & 7) != 0)
        return -1;
    const Kv8Parts parts{part_o, part_ml, splits, token_req == nullptr ? qo_indptr + first_entry : nullptr, count};
    const Kv8AttnArgs a{q, out, (const uint8_t*)codes, (const uint8_t*)scales, block_table, qo_indptr, kv_len, token_req,
                        cache_pos, q_stride, bt_stride, pages, nq, nkv, hd, window, keep_first, first_entry, scale,
                        page_split(page_size), parts};
    const long long rows = (long long)max_q * (nq / nkv);
    const int R = rows <= 8 ? 8 : 64;
    const long long tiles = (rows + R - 1) / R;
    if (tiles > 65535) return -1;
    const dim3 grid(nkv * splits, (unsigned)tiles, count);
    const cudaStream_t s = (cudaStream_t)stream;
    int code;
    if (act_dtype == MSTAR_F32) code = R == 8 ? launch_simt<float, 8>(a, grid, s) : launch_simt<float, 64>(a, grid, s);
    else code = R == 8 ? launch_simt<bf16, 8>(a, grid, s) : launch_simt<bf16, 64>(a, grid, s);
    if (code != 0 || splits == 1) return code;
    return kv8_merge(parts, out, act_dtype, tokens, nq, hd, s);
}

MSTAR_API int mstar_kv8_attention_packed(const long long* a) {
    return mstar_kv8_attention((const void*)a[0], (int)a[1], (void*)a[2], (int)a[3], (const void*)a[4],
        (const void*)a[5], (int)a[6], (const int*)a[7], (int)a[8], (const int*)a[9], (const int*)a[10],
        (const int*)a[11], (const int*)a[12], (int)a[13], (int)a[14], (int)a[15], (int)a[16], (int)a[17], (int)a[18],
        (int)a[19], (int)a[20], (int)a[21], (int)a[22], kv8_packed_float(a[23]), (int)a[24], (float*)a[25],
        (float*)a[26], (void*)a[27]);
}
