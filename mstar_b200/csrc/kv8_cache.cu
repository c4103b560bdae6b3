// Writing the 8-bit cache and reading rows back (format: kv8.cuh).
//
// mstar_rope_kv8_write: one block per token and slice of its heads; 8 features a thread, the threads of a head side
// by side in a warp.  Queries and keys are rotated, keys and values are quantised: the row's largest number by
// shuffles, the codes as one 8-byte store a thread, the scale byte by the first one.  The rotated queries go to a
// tensor of their own, so that the projection's output stays as it was and the attention after it reads rows without
// gaps.
//
// Angles: position * frequency is exact in double (24 + 24 bits), is taken to half-turns and brought into [-1, 1]
// there, so that far positions lose nothing (in float, position 100,000 would be off by 0.004).  In the 16-bit mode
// sine and cosine of the remainder and the rotation are float; in the 32-bit mode both are double, since a key next
// to the border of two codes would be off by a whole code: 1/16 of its value.
//
// The reference's cache has no 8-bit form (mstar/engine/kv_cache_engine.py:132-136).
#include "kv8.cuh"

struct Kv8WriteArgs {
    const int *positions, *cache_pos, *token_req, *block_table;
    const float* inv_freq;
    uint8_t *codes, *scales;
    int nq, nkv, hd, rot, interleaved, bt_stride, pages, in_stride;
    PageSplit page;
};

// 8 of row[d ..] as floats; V: the row is aligned to 8 elements
template <bool V, typename A> __device__ __forceinline__ void take8(const A* p, float (&x)[8]) {
    if constexpr (V) {
        load8(p, x);
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) x[i] = to_float(p[i]);
    }
}

// R: the type of the rotation, float or double
__device__ __forceinline__ void half_turns(float t, float* sn, float* cs) { sincospif(t, sn, cs); }
__device__ __forceinline__ void half_turns(double t, double* sn, double* cs) { sincospi(t, sn, cs); }

// L: threads of a head, a power of two with 8 L >= hd.  V: pairs, halves and rows in whole aligned groups of 8.
template <typename A, typename R, int L, bool V>
__global__ void __launch_bounds__(256) rope_kv8_write_kernel(const A* __restrict__ qkv, A* __restrict__ q_out,
                                                             Kv8WriteArgs a) {
    pdl_launch_dependents();   // a short kernel: the long one after it may be scheduled now
    qkv = pdl_after(qkv, pdl_wait());
    __shared__ R tab_sn[128], tab_cs[128];
    const int t = blockIdx.x, hd = a.hd, half = a.rot >> 1;
    for (int j = threadIdx.x; j < half; j += blockDim.x) {
        double turns = (double)a.positions[t] * (double)a.inv_freq[j] * 0.31830988618379067154;   // half-turns
        turns -= 2.0 * rint(0.5 * turns);
        half_turns((R)turns, &tab_sn[j], &tab_cs[j]);
    }
    const int cp = a.cache_pos[t], logical = cp < 0 ? -1 : page_of(a.page, cp);
    int page = -1;
    if (logical >= 0 && logical < a.bt_stride) page = a.block_table[(size_t)a.token_req[t] * a.bt_stride + logical];
    const bool held = page >= 0 && page < a.pages;
    const int slot = held ? cp - logical * a.page.size : 0;
    __syncthreads();

    constexpr int PER = 256 / L;
    const int l = threadIdx.x % L, d0 = l * 8;
    const bool in = d0 < hd;
    const int heads = a.nq + 2 * a.nkv;
    const A* row = qkv + (size_t)t * a.in_stride;
    for (int h = blockIdx.y * PER + threadIdx.x / L; h < heads; h += gridDim.y * PER) {
        float y[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) y[i] = 0.f;
        if (in) {
            const A* src = row + (size_t)h * hd;
            take8<V>(src + d0, y);
            if (h < a.nq + a.nkv && d0 < a.rot) {
                if (V && a.interleaved) {
#pragma unroll
                    for (int i = 0; i < 8; i += 2) {
                        const R sn = tab_sn[(d0 + i) >> 1], cs = tab_cs[(d0 + i) >> 1];
                        const R x0 = y[i], x1 = y[i + 1];
                        y[i] = (float)(x0 * cs - x1 * sn);
                        y[i + 1] = (float)(x1 * cs + x0 * sn);
                    }
                } else if (V) {
                    const bool upper = d0 >= half;
                    const int j0 = upper ? d0 - half : d0;
                    float z[8];
                    take8<V>(src + (upper ? d0 - half : d0 + half), z);
#pragma unroll
                    for (int i = 0; i < 8; ++i) {
                        const R sn = upper ? tab_sn[j0 + i] : -tab_sn[j0 + i];
                        y[i] = (float)((R)y[i] * tab_cs[j0 + i] + (R)z[i] * sn);
                    }
                } else {
                    for (int i = 0; i < 8; ++i) {
                        const int d = d0 + i;
                        if (d >= a.rot) break;
                        const bool upper = a.interleaved ? (d & 1) : d >= half;
                        const int j = a.interleaved ? d >> 1 : upper ? d - half : d;
                        const int other = a.interleaved ? d ^ 1 : upper ? d - half : d + half;
                        const R sn = upper ? tab_sn[j] : -tab_sn[j];
                        y[i] = (float)((R)y[i] * tab_cs[j] + (R)to_float(src[other]) * sn);
                    }
                }
            }
        }
        if (h < a.nq) {
            if (in) {
                A* dst = q_out + (size_t)t * a.nq * hd + (size_t)h * hd + d0;
                if constexpr (V) {
                    store8(dst, y);
                } else {
#pragma unroll
                    for (int i = 0; i < 8; ++i) dst[i] = from_float<A>(y[i]);
                }
            }
            continue;                                     // (all threads of a head)
        }
        float most = 0.f;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const float m = fabsf(y[i]);
            most = m < INFINITY ? fmaxf(most, m) : INFINITY;      // (not less for NaN too; stays infinite below)
        }
        // heads of a warp may take part in different numbers of rounds: only this head's threads meet
        const unsigned mask = L == 32 ? 0xffffffffu : ((1u << (L & 31)) - 1u) << ((threadIdx.x & 31) / L * L);
#pragma unroll
        for (int o = L / 2; o > 0; o >>= 1) most = fmaxf(most, __shfl_xor_sync(mask, most, o));
        if (!held) continue;
        const int byte = kv8_scale_byte(most);
        const bool bad = byte == KV8_BAD_BYTE;
        const float inv = kv8_inverse_scale(bad ? 127 : byte);
        const int r = h - a.nq;                           // key heads, then value heads: the order of a page's planes
        const size_t at = ((size_t)page * 2 * a.nkv + r) * a.page.size + slot;
        if (in) {
            const uint2 w = make_uint2(kv8_pack4(y[0] * inv, y[1] * inv, y[2] * inv, y[3] * inv),
                                       kv8_pack4(y[4] * inv, y[5] * inv, y[6] * inv, y[7] * inv));
            *reinterpret_cast<uint2*>(a.codes + at * hd + d0) = bad ? make_uint2(0u, 0u) : w;
        }
        if (l == 0) a.scales[at] = (uint8_t)byte;
    }
}

template <typename A, typename R, int L>
static int launch_write(const void* qkv, void* q_out, const Kv8WriteArgs& a, int tokens, bool vec, cudaStream_t s) {
    const int per = 256 / L, heads = a.nq + 2 * a.nkv;
    int slices = (heads + per - 1) / per;
    if (tokens >= 256) slices = 1;      // enough blocks: a token's angles once
    if (slices > 65535) return -1;
    const dim3 grid(tokens, slices);
    cudaError_t e;
    if (vec) e = mstar_launch((rope_kv8_write_kernel<A, R, L, true>), grid, dim3(256), 0, s, (const A*)qkv, (A*)q_out, a);
    else e = mstar_launch((rope_kv8_write_kernel<A, R, L, false>), grid, dim3(256), 0, s, (const A*)qkv, (A*)q_out, a);
    return e != cudaSuccess ? (int)e : launch_status();
}

// qkv: `tokens` rows of (nq + 2 nkv) * hd elements, `in_stride` apart.  nkv 0: queries only.  hd a multiple of 8, at
// most 256; rot even, at most hd.  Returns 0, a CUDA error code or -1 (shape refused).
MSTAR_API int mstar_rope_kv8_write(const void* qkv, int act_dtype, int in_stride, void* q_out, const int* positions,
                                   const int* cache_pos, const int* token_req, const int* block_table, int bt_stride,
                                   const float* inv_freq, void* codes, void* scales, int pages, int tokens, int nq,
                                   int nkv, int hd, int rot, int interleaved, int page_size, void* stream) {
    if (tokens <= 0) return 0;
    if (hd <= 0 || hd % 8 != 0 || hd > 256 || rot < 0 || rot % 2 != 0 || rot > hd || nq < 0 || nkv < 0 || page_size <= 0 ||
        pages <= 0 || ((uintptr_t)codes & 7) != 0)
        return -1;
    const Kv8WriteArgs a{positions, cache_pos, token_req, block_table, inv_freq, (uint8_t*)codes, (uint8_t*)scales, nq,
                         nkv, hd, rot, interleaved, bt_stride, pages, in_stride, page_split(page_size)};
    const int item = act_dtype == MSTAR_F32 ? 4 : 2;
    const bool vec = (interleaved ? rot % 8 == 0 : rot % 16 == 0) && ((uintptr_t)qkv & 15) == 0 &&
                     ((uintptr_t)q_out & 15) == 0 && (in_stride * item) % 16 == 0;
    const cudaStream_t s = (cudaStream_t)stream;
    if (act_dtype == MSTAR_F32) {
        if (hd <= 64) return launch_write<float, double, 8>(qkv, q_out, a, tokens, vec, s);
        if (hd <= 128) return launch_write<float, double, 16>(qkv, q_out, a, tokens, vec, s);
        return launch_write<float, double, 32>(qkv, q_out, a, tokens, vec, s);
    }
    if (hd <= 64) return launch_write<bf16, float, 8>(qkv, q_out, a, tokens, vec, s);
    if (hd <= 128) return launch_write<bf16, float, 16>(qkv, q_out, a, tokens, vec, s);
    return launch_write<bf16, float, 32>(qkv, q_out, a, tokens, vec, s);
}

// ------------------------------------------------------------------------------- rows read back
// 8 features a thread and U such runs, 256 apart, whose chains of loads (place, table entry, codes) go side by side: a
// run alone is three latencies for 24 bytes.
struct Kv8ReadArgs {
    const uint8_t *codes, *scales;
    const int *block_table, *token_req, *cache_pos;
    int bt_stride, rows, hd, pages, runs;
    PageSplit page, per_row, per_token;      // runs of a row, runs of a token
};
template <typename A, int U> __global__ void __launch_bounds__(256) kv8_read_rows_kernel(Kv8ReadArgs a, A* out) {
    pdl_launch_dependents();
    pdl_wait();
    const int first = blockIdx.x * (256 * U) + threadIdx.x;
    int t[U], cp[U], id[U], req[U];
    size_t at[U];
    int d[U], scale[U];
    uint2 w[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
        const int run = min(first + u * 256, a.runs - 1);
        t[u] = page_of(a.per_token, run);
        cp[u] = a.cache_pos[t[u]];
        req[u] = a.token_req[t[u]];
        d[u] = run - t[u] * a.per_token.size;
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
        const int logical = cp[u] < 0 ? -1 : page_of(a.page, cp[u]);
        id[u] = logical >= 0 && logical < a.bt_stride ? a.block_table[(size_t)req[u] * a.bt_stride + logical] : -1;
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
        const int r = page_of(a.per_row, d[u]);
        d[u] = (d[u] - r * a.per_row.size) * 8;
        const bool held = id[u] >= 0 && id[u] < a.pages;
        const int slot = held ? cp[u] - page_of(a.page, cp[u]) * a.page.size : 0;
        at[u] = ((size_t)(held ? id[u] : 0) * a.rows + r) * a.page.size + slot;
        w[u] = held ? *reinterpret_cast<const uint2*>(a.codes + at[u] * a.hd + d[u]) : make_uint2(0u, 0u);
        scale[u] = held ? a.scales[at[u]] : 0;
        at[u] = ((size_t)t[u] * a.rows + r) * a.hd + d[u];
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
        if (first + u * 256 >= a.runs) break;
        const float s = kv8_scale(scale[u]);
        float v[8];
        kv8_unpack4(w[u].x, v);
        kv8_unpack4(w[u].y, v + 4);
#pragma unroll
        for (int k = 0; k < 8; ++k) v[k] *= s;
        store8(out + at[u], v);
    }
}

template <typename A>
static cudaError_t launch_read(const Kv8ReadArgs& a, void* out, cudaStream_t s) {
    // four runs a thread where they still give every SM two blocks (16,000 tokens' 16 rows of 128: 20.8 us, with a block
    // a token 34.1); one where they are few (11 tokens' rows: 1.4 us)
    const int blocks = (a.runs + 255) / 256;
    if (blocks >= 8 * device_sm_count())
        return mstar_launch((kv8_read_rows_kernel<A, 4>), dim3((blocks + 3) / 4), dim3(256), 0, s, a, (A*)out);
    return mstar_launch((kv8_read_rows_kernel<A, 1>), dim3(blocks), dim3(256), 0, s, a, (A*)out);
}

// out [tokens, 2, nkv, hd]: the rows of the given tokens; zeros where the table has no page.  hd a multiple of 8.
MSTAR_API int mstar_kv8_read_rows(const void* codes, const void* scales, const int* block_table, int bt_stride,
                                  const int* token_req, const int* cache_pos, void* out, int out_dtype, int tokens,
                                  int nkv, int hd, int pages, int page_size, void* stream) {
    if (tokens <= 0) return 0;
    if (hd <= 0 || hd % 8 != 0 || nkv <= 0 || page_size <= 0 || pages <= 0 || ((uintptr_t)codes & 7) != 0 ||
        ((uintptr_t)out & 15) != 0)
        return -1;
    const int per_row = hd / 8, rows = 2 * nkv;
    const cudaStream_t s = (cudaStream_t)stream;
    // runs are counted in 31 bits: several launches beyond that
    const int most = (1 << 30) / (rows * per_row);
    if (most < 1) return -1;
    cudaError_t e = cudaSuccess;
    for (long long t0 = 0; t0 < tokens && e == cudaSuccess; t0 += most) {
        const int n = tokens - t0 < most ? (int)(tokens - t0) : most;
        const Kv8ReadArgs a{(const uint8_t*)codes, (const uint8_t*)scales, block_table, token_req + t0, cache_pos + t0,
                            bt_stride, rows, hd, pages, n * rows * per_row, page_split(page_size), page_split(per_row),
                            page_split(rows * per_row)};
        const size_t at = (size_t)t0 * rows * hd;
        e = out_dtype == MSTAR_F32 ? launch_read<float>(a, (float*)out + at, s) : launch_read<bf16>(a, (bf16*)out + at, s);
    }
    return e != cudaSuccess ? (int)e : launch_status();
}

MSTAR_API int mstar_rope_kv8_write_packed(const long long* a) {
    return mstar_rope_kv8_write((const void*)a[0], (int)a[1], (int)a[2], (void*)a[3], (const int*)a[4],
        (const int*)a[5], (const int*)a[6], (const int*)a[7], (int)a[8], (const float*)a[9], (void*)a[10],
        (void*)a[11], (int)a[12], (int)a[13], (int)a[14], (int)a[15], (int)a[16], (int)a[17], (int)a[18], (int)a[19],
        (void*)a[20]);
}
MSTAR_API int mstar_kv8_read_rows_packed(const long long* a) {
    return mstar_kv8_read_rows((const void*)a[0], (const void*)a[1], (const int*)a[2], (int)a[3], (const int*)a[4],
        (const int*)a[5], (void*)a[6], (int)a[7], (int)a[8], (int)a[9], (int)a[10], (int)a[11], (int)a[12],
        (void*)a[13]);
}
