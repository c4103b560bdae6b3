// Writing the 8-bit cache and reading rows back (format: kv8.cuh).
//
// mstar_rope_kv8_write: a block per token (or part of its heads).  A thread has 16 features of a head, 8 and the 8 that they
// are turned with, so that every number is read once, and the threads of a head lie side by side in a warp: the row's largest
// number comes by shuffles, codes go out as 8-byte stores, the scale byte by the first thread.  The loads go before the
// angles, whose latency they share.  The rotated queries go to a tensor of their own, so that the projection's output stays
// as it was and the attention after it reads rows without gaps.
//
// Angles: position * frequency is exact in double (24 + 24 bits), is taken to half-turns (off by less than 2^-52 of the angle)
// and brought into [-1, 1] there (in float, position 100,000 would be off by 0.004; here by 2^-35).  A key next to the border of
// two codes that came out on the wrong side would be off by a whole code, 1/16 of its value (with a rotation in float one
// number in some 10^6), so sines and cosines are double, and the rotation is too in the 32-bit mode.  In the 16-bit mode it
// is done in pairs of floats: c = c_hi + c_lo with 16 bits in c_hi, so that its product with a bfloat16 is exact, the two
// products are added with the sum's rounding error (Knuth's two-sum), and the small parts are added to that.
//
// 2,048 tokens of 24 + 16 heads of 128 take 11.2 us for 38 MB (5.8 at the copy bandwidth), 999 float tokens of 48 heads of
// 64 5.0: bound by the latency of a block's chain (position, sines in double, rotation, largest number), of which few
// an SM run at a time.  Threads with 8 features that read their partners' too, heads one after another, took 11.2
// with a rotation in float, 14.9 with the keys' in double; the next head's loads ahead, 13.3.
//
// The reference's cache has no 8-bit form (mstar/engine/kv_cache_engine.py:132-136).
#include "kv8.cuh"

struct Kv8WriteArgs {
    const int *positions, *cache_pos, *token_req, *block_table;
    const float* inv_freq;
    uint8_t *codes, *scales;
    int nq, nkv, hd, rot, interleaved, bt_stride, bt_width, pages, in_stride;
    PageSplit page;
};

// 8 features as they are loaded: one or two 16-byte words
template <typename A> struct Run8 { uint4 w[sizeof(A) / 2]; };
__device__ __forceinline__ void numbers(const Run8<bf16>& r, float (&x)[8]) {
    const __nv_bfloat162* h = reinterpret_cast<const __nv_bfloat162*>(&r);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float2 f = __bfloat1622float2(h[i]);
        x[2 * i] = f.x;
        x[2 * i + 1] = f.y;
    }
}
__device__ __forceinline__ void numbers(const Run8<float>& r, float (&x)[8]) {
    const float* f = reinterpret_cast<const float*>(&r);
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = f[i];
}
// two floats side by side
__device__ __forceinline__ uint64_t two(float a, float b) {
    return (uint64_t)__float_as_uint(a) | ((uint64_t)__float_as_uint(b) << 32);
}
__device__ __forceinline__ float first(uint64_t x) { return __uint_as_float((uint32_t)x); }
__device__ __forceinline__ float second(uint64_t x) { return __uint_as_float((uint32_t)(x >> 32)); }
__device__ __forceinline__ uint64_t mul2(uint64_t a, uint64_t b) {
    uint64_t r;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
    uint64_t r;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
    uint64_t r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
    return r;
}
// x c + z s, c and s in two parts: to within some 2^-38 of the products, then rounded once.  A sum that is not finite stays
// so (its rounding error, inf - inf, makes it NaN: what is held as NaNs either way).
__device__ __forceinline__ uint64_t turned(uint64_t x, uint64_t z, uint64_t ch, uint64_t cl, uint64_t sh, uint64_t sl) {
    const uint64_t less = two(-1.f, -1.f);
    const uint64_t p = mul2(x, ch), q = mul2(z, sh), sum = add2(p, q), b = fma2(p, less, sum);
    const uint64_t e = add2(fma2(fma2(b, less, sum), less, p), fma2(b, less, q));
    return add2(sum, fma2(z, sl, fma2(x, cl, e)));
}

// L: threads of a head, a power of two with 16 L >= hd.  V: rows in whole aligned groups of 16, turned in groups of 8.
template <typename A, int L, bool V>
__global__ void __launch_bounds__(512) rope_kv8_write_kernel(const A* qkv, A* q_out, Kv8WriteArgs a) {
    pdl_launch_dependents();   // a short kernel: the long one after it may be scheduled now
    pdl_wait();
    constexpr bool PARTS = V && sizeof(A) == 2;
    __shared__ double sn_d[PARTS ? 1 : 128], cs_d[PARTS ? 1 : 128];
    __shared__ __align__(16) float sh_t[PARTS ? 128 : 1], sl_t[PARTS ? 128 : 1], ch_t[PARTS ? 128 : 1], cl_t[PARTS ? 128 : 1];
    const int t = blockIdx.x, hd = a.hd, half = a.rot >> 1, heads = a.nq + 2 * a.nkv;
    const int h = blockIdx.y * (blockDim.x / L) + threadIdx.x / L, u = threadIdx.x % L;
    // the thread's features: d[0] .. and d[1] .., rotated ones with their partners
    int d[2] = {16 * u, 16 * u + 8};
    if (V && !a.interleaved) {
        const int turns = a.rot >> 4;
        d[0] = u < turns ? 8 * u : a.rot + 8 * (u - turns);
        d[1] = d[0] + (u < turns ? half : (hd - a.rot) >> 1);
    }
    const A* src = qkv + (size_t)t * a.in_stride + (size_t)h * hd;
    const bool in = h < heads && 16 * u < hd;
    Run8<A> own[2];
    if (V && in) {
#pragma unroll
        for (int k = 0; k < 2; ++k) own[k] = *reinterpret_cast<const Run8<A>*>(src + d[k]);
    }
    const int cp = a.cache_pos[t], req = a.token_req[t];
    const int logical = cp < 0 ? -1 : page_of(a.page, cp);
    int page = -1;
    if (logical >= 0 && logical < a.bt_width) page = a.block_table[(size_t)req * a.bt_stride + logical];
    for (int j = threadIdx.x; j < half; j += blockDim.x) {
        double turns = (double)a.positions[t] * (double)a.inv_freq[j] * 0.31830988618379067154, sn, cs;   // half-turns
        turns -= 2.0 * rint(0.5 * turns);
        sincospi(turns, &sn, &cs);
        if constexpr (PARTS) {
            // (the last 8 of 24 bits cut off)
            sh_t[j] = __uint_as_float(__float_as_uint((float)sn) & 0xffffff00u);
            ch_t[j] = __uint_as_float(__float_as_uint((float)cs) & 0xffffff00u);
            sl_t[j] = (float)(sn - (double)sh_t[j]);
            cl_t[j] = (float)(cs - (double)ch_t[j]);
        } else {
            sn_d[j] = sn;
            cs_d[j] = cs;
        }
    }
    const bool held = page >= 0 && page < a.pages;
    const int slot = held ? cp - logical * a.page.size : 0;
    __syncthreads();
    if (h >= heads) return;

    float y[2][8];
#pragma unroll
    for (int k = 0; k < 2; ++k)
#pragma unroll
        for (int i = 0; i < 8; ++i) y[k][i] = 0.f;
    if (in) {
        const bool turn = h < a.nq + a.nkv && (V && !a.interleaved ? 16 * u : d[0]) < a.rot;
        if constexpr (V) {
            numbers(own[0], y[0]);
            numbers(own[1], y[1]);
            if (turn && !a.interleaved) {
#pragma unroll
                for (int i = 0; i < 8; i += 2) {
                    const int j = d[0] + i;
                    if constexpr (PARTS) {
                        const uint64_t ch = *reinterpret_cast<const uint64_t*>(ch_t + j), cl = *reinterpret_cast<const uint64_t*>(cl_t + j);
                        const uint64_t sh = *reinterpret_cast<const uint64_t*>(sh_t + j), sl = *reinterpret_cast<const uint64_t*>(sl_t + j);
                        const uint64_t x = two(y[0][i], y[0][i + 1]), z = two(y[1][i], y[1][i + 1]);
                        const uint64_t lo = turned(x, two(-y[1][i], -y[1][i + 1]), ch, cl, sh, sl), up = turned(z, x, ch, cl, sh, sl);
                        y[0][i] = first(lo);
                        y[0][i + 1] = second(lo);
                        y[1][i] = first(up);
                        y[1][i + 1] = second(up);
                    } else {
#pragma unroll
                        for (int k = 0; k < 2; ++k) {
                            const double sn = sn_d[j + k], cs = cs_d[j + k], x = y[0][i + k], z = y[1][i + k];
                            y[0][i + k] = (float)(x * cs - z * sn);
                            y[1][i + k] = (float)(z * cs + x * sn);
                        }
                    }
                }
            } else if (turn) {
#pragma unroll
                for (int k = 0; k < 2; ++k)
#pragma unroll
                    for (int i = 0; i < 8; i += 2) {
                        const int j = (d[k] + i) >> 1;
                        const float x = y[k][i], z = y[k][i + 1];
                        if constexpr (PARTS) {
                            const uint64_t r = turned(two(x, z), two(-z, x), two(ch_t[j], ch_t[j]), two(cl_t[j], cl_t[j]),
                                                      two(sh_t[j], sh_t[j]), two(sl_t[j], sl_t[j]));
                            y[k][i] = first(r);
                            y[k][i + 1] = second(r);
                        } else {
                            const double sn = sn_d[j], cs = cs_d[j];
                            y[k][i] = (float)(x * cs - z * sn);
                            y[k][i + 1] = (float)(z * cs + x * sn);
                        }
                    }
            }
        } else {
#pragma unroll
            for (int k = 0; k < 2; ++k)
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    const int at = d[k] + i;
                    if (at >= hd) break;
                    y[k][i] = to_float(src[at]);
                    if (h < a.nq + a.nkv && at < a.rot) {
                        const bool upper = a.interleaved ? (at & 1) : at >= half;
                        const int j = a.interleaved ? at >> 1 : upper ? at - half : at;
                        const int other = a.interleaved ? at ^ 1 : upper ? at - half : at + half;
                        const double sn = upper ? sn_d[j] : -sn_d[j];
                        y[k][i] = (float)((double)y[k][i] * cs_d[j] + (double)to_float(src[other]) * sn);
                    }
                }
        }
    }
    if (h < a.nq) {
        if (in) {
            A* dst = q_out + (size_t)t * a.nq * hd + (size_t)h * hd;
#pragma unroll
            for (int k = 0; k < 2; ++k) {
                if constexpr (V) {
                    store8(dst + d[k], y[k]);
                } else {
#pragma unroll
                    for (int i = 0; i < 8; ++i)
                        if (d[k] + i < hd) dst[d[k] + i] = from_float<A>(y[k][i]);
                }
            }
        }
        return;                                           // (all threads of a head)
    }
    float most = 0.f;
#pragma unroll
    for (int k = 0; k < 2; ++k)
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const float m = fabsf(y[k][i]);
            most = m < INFINITY ? fmaxf(most, m) : INFINITY;      // (not less for NaN too; stays infinite below)
        }
    // other heads of the warp may have left: only this head's threads meet
    const unsigned mask = ((1u << L) - 1u) << ((threadIdx.x & 31) / L * L);
#pragma unroll
    for (int o = L / 2; o > 0; o >>= 1) most = fmaxf(most, __shfl_xor_sync(mask, most, o));
    if (!held) return;
    const int byte = kv8_scale_byte(most);
    const bool bad = byte == KV8_BAD_BYTE;
    const float inv = kv8_inverse_scale(bad ? 127 : byte);
    const int r = h - a.nq;                               // key heads, then value heads: the order of a page's planes
    const size_t at = ((size_t)page * 2 * a.nkv + r) * a.page.size + slot;
#pragma unroll
    for (int k = 0; k < 2; ++k)
        if (in && d[k] < hd) {
            const uint2 w = make_uint2(kv8_pack4(y[k][0] * inv, y[k][1] * inv, y[k][2] * inv, y[k][3] * inv),
                                       kv8_pack4(y[k][4] * inv, y[k][5] * inv, y[k][6] * inv, y[k][7] * inv));
            *reinterpret_cast<uint2*>(a.codes + at * hd + d[k]) = bad ? make_uint2(0u, 0u) : w;
        }
    if (u == 0) a.scales[at] = (uint8_t)byte;
}

template <typename A, int L>
static int launch_write(const void* qkv, void* q_out, const Kv8WriteArgs& a, int tokens, bool vec, cudaStream_t s) {
    // A token's heads in one block in the 32-bit mode, so that its angles are made once; in two in the 16-bit mode, which
    // leaves more blocks whose chains overlap (2,048 and 512 tokens of 40 heads of 128: 11.2 and 3.7 us, 12.5 and 5.1 in one,
    // 12.2 and 4.4 in three; 999 float tokens 5.0 in one and 5.6 in two).  With few tokens in blocks of 128 threads.
    const long long all = (long long)(a.nq + 2 * a.nkv) * L, part = sizeof(A) == 2 ? (all + 1) / 2 : all;
    const int threads = tokens < 256 ? 128 : (int)min(512ll, (part + 31) / 32 * 32);
    const long long slices = (all + threads - 1) / threads;
    if (slices > 65535) return -1;
    const dim3 grid(tokens, (unsigned)slices);
    cudaError_t e;
    if (vec) e = mstar_launch((rope_kv8_write_kernel<A, L, true>), grid, dim3(threads), 0, s, (const A*)qkv, (A*)q_out, a);
    else e = mstar_launch((rope_kv8_write_kernel<A, L, false>), grid, dim3(threads), 0, s, (const A*)qkv, (A*)q_out, a);
    return e != cudaSuccess ? (int)e : launch_status();
}

// qkv: `tokens` rows of (nq + 2 nkv) * hd elements, `in_stride` apart.  hd a multiple of 8, at most 256; rot even, at most
// hd.  Returns 0, a CUDA error code or -1 (shape refused).
MSTAR_API int mstar_rope_kv8_write(const void* qkv, int act_dtype, int in_stride, void* q_out, const int* positions,
                                   const int* cache_pos, const int* token_req, const int* block_table, int bt_stride,
                                   int bt_width, const float* inv_freq, void* codes, void* scales, int pages, int tokens, int nq,
                                   int nkv, int hd, int rot, int interleaved, int page_size, void* stream) {
    if (tokens <= 0) return 0;
    if (hd <= 0 || hd % 8 != 0 || hd > 256 || rot < 0 || rot % 2 != 0 || rot > hd || nq <= 0 || nkv <= 0 || page_size <= 0 ||
        pages <= 0 || ((uintptr_t)codes & 7) != 0)
        return -1;
    const Kv8WriteArgs a{positions, cache_pos, token_req, block_table, inv_freq, (uint8_t*)codes, (uint8_t*)scales, nq,
                         nkv, hd, rot, interleaved, bt_stride, bt_width, pages, in_stride, page_split(page_size)};
    const int item = act_dtype == MSTAR_F32 ? 4 : 2;
    const bool vec = hd % 16 == 0 && rot % 16 == 0 && ((uintptr_t)qkv & 15) == 0 && ((uintptr_t)q_out & 15) == 0 &&
                     (in_stride * item) % 16 == 0;
    const cudaStream_t s = (cudaStream_t)stream;
    if (act_dtype == MSTAR_F32) {
        if (hd <= 64) return launch_write<float, 4>(qkv, q_out, a, tokens, vec, s);
        if (hd <= 128) return launch_write<float, 8>(qkv, q_out, a, tokens, vec, s);
        return launch_write<float, 16>(qkv, q_out, a, tokens, vec, s);
    }
    if (hd <= 64) return launch_write<bf16, 4>(qkv, q_out, a, tokens, vec, s);
    if (hd <= 128) return launch_write<bf16, 8>(qkv, q_out, a, tokens, vec, s);
    return launch_write<bf16, 16>(qkv, q_out, a, tokens, vec, s);
}

// ------------------------------------------------------------------------------- rows read back
// 8 features a thread and U such runs, 256 apart, whose chains of loads (place, table entry, codes) go side by side: a
// run alone is three latencies for 24 bytes.
struct Kv8ReadArgs {
    const uint8_t *codes, *scales;
    const int *block_table, *token_req, *cache_pos;
    int bt_stride, bt_width, rows, hd, pages, runs;
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
        id[u] = logical >= 0 && logical < a.bt_width ? a.block_table[(size_t)req[u] * a.bt_stride + logical] : -1;
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
        // (streaming stores: what is read again soonest are the codes; 16,000 tokens' rows 18.7 us, 19.8 without)
        Run8<A> r;
        store8(reinterpret_cast<A*>(r.w), v);
#pragma unroll
        for (int k = 0; k < (int)sizeof(A) / 2; ++k) __stcs(reinterpret_cast<uint4*>(out + at[u]) + k, r.w[k]);
    }
}

template <typename A>
static cudaError_t launch_read(const Kv8ReadArgs& a, void* out, cudaStream_t s) {
    // two runs a thread where they still give every SM four blocks (16,000 tokens' 16 rows of 128: 18.7 us, with four runs
    // 19.1, with a block a token 34.1; 2,000 tokens' 3.5, 4.6 with four); one where they are few (11 tokens' rows: 1.4 us)
    const int blocks = (a.runs + 255) / 256;
    if (blocks >= 8 * device_sm_count())
        return mstar_launch((kv8_read_rows_kernel<A, 2>), dim3((blocks + 1) / 2), dim3(256), 0, s, a, (A*)out);
    return mstar_launch((kv8_read_rows_kernel<A, 1>), dim3(blocks), dim3(256), 0, s, a, (A*)out);
}

// out [tokens, 2, nkv, hd]: the rows of the given tokens; zeros where the table has no page.  hd a multiple of 8.
MSTAR_API int mstar_kv8_read_rows(const void* codes, const void* scales, const int* block_table, int bt_stride,
                                  int bt_width, const int* token_req, const int* cache_pos, void* out, int out_dtype, int tokens,
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
                            bt_stride, bt_width, rows, hd, pages, n * rows * per_row, page_split(page_size), page_split(per_row),
                            page_split(rows * per_row)};
        const size_t at = (size_t)t0 * rows * hd;
        e = out_dtype == MSTAR_F32 ? launch_read<float>(a, (float*)out + at, s) : launch_read<bf16>(a, (bf16*)out + at, s);
    }
    return e != cudaSuccess ? (int)e : launch_status();
}

MSTAR_API int mstar_rope_kv8_write_packed(const long long* a) {
    return mstar_rope_kv8_write((const void*)a[0], (int)a[1], (int)a[2], (void*)a[3], (const int*)a[4],
        (const int*)a[5], (const int*)a[6], (const int*)a[7], (int)a[8], (int)a[9], (const float*)a[10], (void*)a[11],
        (void*)a[12], (int)a[13], (int)a[14], (int)a[15], (int)a[16], (int)a[17], (int)a[18], (int)a[19], (int)a[20],
        (void*)a[21]);
}
MSTAR_API int mstar_kv8_read_rows_packed(const long long* a) {
    return mstar_kv8_read_rows((const void*)a[0], (const void*)a[1], (const int*)a[2], (int)a[3], (int)a[4], (const int*)a[5],
        (const int*)a[6], (void*)a[7], (int)a[8], (int)a[9], (int)a[10], (int)a[11], (int)a[12], (int)a[13],
        (void*)a[14]);
}
