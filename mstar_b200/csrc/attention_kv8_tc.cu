// Attention of prompt portions over the 8-bit cache (format: kv8.cuh) on the fifth-generation tensor cores, bfloat16,
// head_dim 64 or 128, up to 128 query heads per kv head, any page size, window and kept first keys.
//
// One CTA owns two row tiles of 128 / G whole tokens each (G query heads per kv head; rows are (token, head) pairs) and
// one kv head, and walks the keys that some of its rows see, 128 at a time.  Its sixteen warps:
//   * 3 warps find a tile's rows through the table (two tiles ahead), and copy its key codes into the tile that the MMAs
//     read (cp.async);
//   * 4 warps read its value codes into registers (the next tile's loads are under way meanwhile), make bfloat16 of them
//     and store the swizzled tile;
//   * one warp issues the products: S_A = Q_A K^T, S_B = Q_B K^T of the next tile as soon as a tile's weights have been
//     used, and O_A += P_A V, O_B += P_B V as soon as weights are there, so that the tensor cores work for one row tile
//     while the other one's softmax runs;
//   * 4 + 4 softmax warps own a row a thread: they read it from tensor memory, keep the running maximum and sum in
//     registers, and write the weights as bfloat16 over the scores (tcgen05.st); the output in tensor memory is rescaled
//     only when a maximum grew by more than 2^8.
// Where the portions have one row tile only and the keys are many, A and B are the same rows, A with the even and B with
// the odd tiles of keys, and their outputs two parts to be joined: 1.4 us a tile instead of 2, for twice the parts.  The
// values' loaders then have three tiles on their way in shared memory instead of one in registers (40.9 us for two
// portions of 17 tokens on 20,000 keys, 42.6 without; with row tiles that differ, 588 instead of 568 below).
//
// What else was built: two buffers of 64 keys a row tile in the same tensor memory, so that scores are made ahead (601 us
// for 2,048 tokens on 14,336 keys, when this took 565: products of 64 keys read the queries from shared memory twice as
// often); the same with two threads a row, which take its steps in turn (571: the exponentials are the same); half a row a
// thread (754: the halves have to meet at every tile); an eighth, a quarter or a third of the exponentials by a polynomial
// (571, 632, 660 when this took 558); one power of two for all queries of a CTA, folded into the keys' factors, so that the
// scores take one product less (565).  What the softmax lacks is neither: its steps wait for one another.
// Tensor memory: S / P 2 x 128 columns, O 2 x head_dim.  Shared memory (head_dim 128): queries 64 KB, two stages of keys
// of 16 KB and two of values of 32 KB each.
//
// The scores' product takes the keys' codes as they are: kind::f8f6f4 at twice the rate of 16-bit operands, and the
// query in two codes, x = hi + lo, so that the two products cost what one of 16 bits does and the keys need neither
// conversion nor a second copy.  A row of queries is scaled by a power of two to have its largest number in (224, 448];
// hi is within 2^-4 of a number, lo leaves 2^-10 at most, 2^-17.8 of the row's largest (a bfloat16 query is within 2^-9
// of itself to begin with).  The keys' scales are a factor a score, two at a time (mul.f32x2); it is NaN for a row that
// is held as NaNs, so that who sees it gets NaNs and nobody else.
//
// Values become bfloat16 with their row's scale folded in, which is exact for every scale: sign, exponent and mantissa
// of a code are moved to bfloat16's places (which reads as the code times 2^-120, subnormal codes included), and a
// product by 2^(120 + e) puts it right (two for e > 7); the even and the odd codes of a word become a pair each, and the
// output's features are put back in order as they are stored.  (float16 values relative to a common exponent need a
// third of the instructions, but rows of values 2^20 apart in size lost the smaller ones.)
//
// What bounds it: per tile of 128 keys and 256 rows (head_dim 128) the MMAs take 2,048 clocks, the exponentials 2,048 (16
// a clock and SM), reading operands and storing tiles some 240 KB of shared memory at 128 bytes a clock; a tile takes
// 4,000, since a row tile's products and its softmax follow one another and the two row tiles share the units.  2,048
// tokens of 32 heads on 16,384 keys: 555 us, 928 TFLOP/s.  Around the tiles a block spends some 12,000 clocks: barriers and
// the first rows 3,000, queries 6,000, outputs 4,000; 2,048 tokens without a cache take 46.7 us, of which the longest
// block's sixteen tiles are 36.
//
// Few row tiles and many keys: the tiles are cut into `splits` ranges whose (maximum, sum, output) go to scratch memory
// and are joined by a second kernel (kv8_merge.cuh).  Row tiles with the most keys are launched first.
//
// Every mbarrier wait is bounded; one that runs out sets the error word (31 to 36) and everybody leaves.
#include "attention_tc_util.cuh"
#include "kv8_merge.cuh"
#include "mma_util.cuh"
#include "tma_util.cuh"

#define K8_ROWS 128
#define K8_KEYS 128
#define K8_THREADS 512
#define K8_SLACK 8.0f
#define K8_AHEAD 3          // PAIR: tiles of values that are asked for before they are used

struct Kv8TcArgs {
    const bf16* q;
    bf16* out;
    const uint8_t *codes, *scales;
    const int *block_table, *qo_indptr, *kv_len;
    int q_stride, bt_stride, bt_width, pages, nq, nkv, window, keep_first, first_entry;
    float scale_log2e;
    PageSplit page;
    Kv8Parts parts;
    int* error_word;
};

__host__ __device__ constexpr int k8_codes(int hd) { return 128 * hd; }          // a tile of codes: 128 rows
__host__ __device__ constexpr int k8_values(int hd) { return K8_KEYS * hd * 2; }
// queries [2 row tiles, PAIR: one][hi, lo], PAIR: values on their way, two stages of keys and of values, of eight tiles each
// key's row, factor and value factor, outputs on their way, the barriers
__host__ __device__ constexpr int k8_smem(int hd, bool pair) {
    return (pair ? 4 + K8_AHEAD : 6) * k8_codes(hd) + 2 * k8_values(hd) + 8 * 128 * 12 + 256 * 128 + 256;
}

template <int R> __device__ __forceinline__ void k8_more_registers() { asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(R)); }
template <int R> __device__ __forceinline__ void k8_less_registers() { asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(R)); }
// Instruction descriptors, D float: kind::f8f6f4 with e4m3 operands, kind::f16 with bfloat16 ones and an MN-major B.
__host__ __device__ constexpr uint32_t k8_idesc_codes(int m, int n) {
    return (1u << 4) | ((uint32_t)(n >> 3) << 17) | ((uint32_t)(m >> 4) << 24);
}
// The products and their commits, issued by the one lane whose `leader` is not zero.  All lanes run the code around them:
// operands computed in a branch of one lane are vector registers, and moving them to uniform ones for every product took
// some 140 clocks a product, twice what the product takes.
__device__ __forceinline__ uint32_t k8_elect() {
    uint32_t r;
    asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(r));
    return r;
}
// (descriptors as their low words, where the address is, beside high words that do not change)
__device__ __forceinline__ void k8_mma_codes(uint32_t leader, uint32_t tmem_d, uint32_t da, uint32_t db, uint32_t high,
                                             uint32_t idesc, uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p, q;\n\t.reg .b64 a, b;\n\t"
        "setp.ne.b32 p, %5, 0;\n\t"
        "setp.ne.b32 q, %6, 0;\n\t"
        "mov.b64 a, {%1, %3};\n\t"
        "mov.b64 b, {%2, %3};\n\t"
        "@q tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], a, b, %4, p;\n\t}"
        ::"r"(tmem_d), "r"(da), "r"(db), "r"(high), "r"(idesc), "r"(accumulate), "r"(leader)
        : "memory");
}
__device__ __forceinline__ void k8_mma_weights(uint32_t leader, uint32_t tmem_d, uint32_t tmem_a, uint32_t db, uint32_t high,
                                               uint32_t idesc, uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p, q;\n\t.reg .b64 b;\n\t"
        "setp.ne.b32 p, %5, 0;\n\t"
        "setp.ne.b32 q, %6, 0;\n\t"
        "mov.b64 b, {%2, %3};\n\t"
        "@q tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], b, %4, p;\n\t}"
        ::"r"(tmem_d), "r"(tmem_a), "r"(db), "r"(high), "r"(idesc), "r"(accumulate), "r"(leader)
        : "memory");
}
__device__ __forceinline__ void k8_commit(uint32_t leader, uint32_t bar) {
    asm volatile(
        "{\n\t.reg .pred q;\n\tsetp.ne.b32 q, %1, 0;\n\t"
        "@q tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n\t}" ::"r"(bar), "r"(leader)
        : "memory");
}
// High words of the descriptors (stride byte offset, version, swizzle) of a tile of codes, K-major: rows of 128 bytes with
// the 128-byte swizzle, or of 64 with the 64-byte one, groups of 8 rows after one another; and of a tile of values.
template <int HD> __host__ __device__ constexpr uint32_t k8_codes_high() {
    return (uint32_t)(8 * HD >> 4) | (1u << 14) | ((HD == 128 ? 2u : 4u) << 29);
}
__host__ __device__ constexpr uint32_t k8_values_high() { return (1024u >> 4) | (1u << 14) | (2u << 29); }
// where a 16-byte run c of row r lies in such a tile
template <int HD> __device__ __forceinline__ uint32_t k8_code_place(int r, int c) {
    return (uint32_t)(r * HD + ((HD == 128 ? c ^ (r & 7) : c ^ ((r >> 1) & 3)) << 4));
}
__device__ __forceinline__ uint64_t k8_two(uint32_t lo, uint32_t hi) { return (uint64_t)lo | ((uint64_t)hi << 32); }
__device__ __forceinline__ uint64_t k8_mul2(uint64_t a, uint64_t b) {
    uint64_t r;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
__device__ __forceinline__ uint64_t k8_fma2(uint64_t a, uint64_t b, uint64_t c) {
    uint64_t r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
    return r;
}
__device__ __forceinline__ uint64_t k8_add2(uint64_t a, uint64_t b) {
    uint64_t r;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
__device__ __forceinline__ float k8_lo(uint64_t x) { return __uint_as_float((uint32_t)x); }
__device__ __forceinline__ float k8_hi(uint64_t x) { return __uint_as_float((uint32_t)(x >> 32)); }
// bits 0 .. n - 1
__device__ __forceinline__ uint32_t k8_below(int n) { return n <= 0 ? 0u : n >= 32 ? 0xffffffffu : (1u << n) - 1u; }

template <int HD, bool PAIR>
__global__ void __launch_bounds__(K8_THREADS, 1) kv8_attention_tc_kernel(Kv8TcArgs a) {
    constexpr int QT = k8_codes(HD), KT = k8_codes(HD), VT = k8_values(HD);
    extern __shared__ __align__(1024) unsigned char smem[];
    unsigned char* q_s = smem;                       // [2 row tiles][hi, lo][128 rows x HD codes]
    constexpr int AHEAD = PAIR ? K8_AHEAD : 0;
    uint4* raw_s = reinterpret_cast<uint4*>(q_s + 2 * QT);           // PAIR: [AHEAD][runs a thread][128 threads] value codes
    unsigned char* k_s = q_s + (PAIR ? 2 + AHEAD : 4) * QT;               // [2 stages][128 keys x HD codes]
    unsigned char* v_s = k_s + 2 * KT;               // [2 stages][HD / 64 blocks][128 keys x 128 bytes]
    // what is told of eight tiles' keys, AHEAD tiles before their keys are copied: tile j + 8's after the scores of tile
    // j + 2 are done, and with them, at the latest, the weights and values of tile j
    uint32_t* row_s = reinterpret_cast<uint32_t*>(v_s + 2 * VT);     // [8][128] rows of the cache
    float* kf_s = reinterpret_cast<float*>(row_s + 1024);            // [8][128] the keys' scales
    uint32_t* vf_s = row_s + 2048;                                   // [8][128] the values' factors
    unsigned char* out_s = reinterpret_cast<unsigned char*>(vf_s + 1024);     // [8 warps][32 rows x 128 bytes] on their way out
    uint64_t* bars = reinterpret_cast<uint64_t*>(out_s + 256 * 128);
    const uint32_t k_full = tc_smem(bars), v_full = tc_smem(bars + 2), k_empty = tc_smem(bars + 4),
                   v_empty = tc_smem(bars + 6), s_full = tc_smem(bars + 8), p_ready = tc_smem(bars + 10),
                   q_ready = tc_smem(bars + 12), o_full = tc_smem(bars + 14), rows_full = tc_smem(bars + 16);
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + 24);

    pdl_wait();
    // PAIR: one row tile, its even and odd key tiles side by side; `splits` ranges of keys, two parts each
    const int splits = PAIR ? a.parts.splits >> 1 : a.parts.splits;
    // (the exchange tells the compiler that a warp has one number: what follows from it need not be kept by every thread)
    const int tid = threadIdx.x, warp = __shfl_sync(0xffffffffu, tid >> 5, 0), lane = tid & 31;
    const int kvh = blockIdx.x / splits, split = blockIdx.x % splits;
    const int e = a.first_entry + blockIdx.z;
    const int G = a.nq / a.nkv, TPT = K8_ROWS / G, RPT = TPT * G;
    const int q_start = a.qo_indptr[e], q_len = a.qo_indptr[e + 1] - q_start;
    const int tok0 = (gridDim.y - 1 - blockIdx.y) * (PAIR ? 1 : 2) * TPT;
    if (tok0 >= q_len) return;
    if ((tc_smem(smem) & 1023u) != 0) {              // the swizzled tiles need this alignment
        if (tid == 0) atomicExch(a.error_word, 31);
        return;
    }
    const int past = a.kv_len[e] - q_len;
    const bool has_b = PAIR || tok0 + TPT < q_len;
    const int last_tok = min(tok0 + (PAIR ? 1 : 2) * TPT, q_len) - 1;
    const SeenKeys seen = seen_keys(past + tok0, past + last_tok, a.window, a.keep_first);
    const int all_tiles = (seen.count + K8_KEYS - 1) / K8_KEYS;
    const int per_split = (all_tiles + splits - 1) / splits;
    const int tile0 = split * per_split, ntiles = max(0, min(all_tiles - tile0, per_split));

    if (tid == 0) {
        for (int i = 0; i < 24; ++i)
            mbar_init(tc_smem(bars + i), i < 2 || i >= 16 ? 96 : i < 4 || i == 12 || i == 13 ? 128 : i == 10 || i == 11 ? 4 : 1);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 12) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(tc_smem(tmem_slot)), "r"(512u)
                     : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    pt_fence_before();
    __syncthreads();
    pt_fence_after();
    const uint32_t tmem = *tmem_slot;

    // what the loaders share: the keys of a tile by their place in it, and the table
    const int* bt = a.block_table + (size_t)e * a.bt_stride;
    const size_t plane = (size_t)a.nkv * a.page.size;
    constexpr int CPR = HD / 16, RP = 128 / CPR;             // 16-byte runs a row, rows of a pass of 128 threads
    if (warp >= 12) {
        // (the launch's 128 a thread, dealt out again: 2 x 184 + 80 + 64 = 512)
        k8_less_registers<64>();
        if (warp > 12) {
            // ------------------------------------------------------------------ rows, factors, keys
            const int kt = tid - 13 * 32;                    // 96 threads; the first 32 have a second key of a tile
            auto entry_of = [&](int j, int c) -> int {
                const int key = key_of(seen, min((tile0 + j) * K8_KEYS + c, seen.count - 1));
                return bt[min(page_of(a.page, key), a.bt_width - 1)];
            };
            auto row_of = [&](int j, int c, int entry) -> uint32_t {
                const int key = key_of(seen, min((tile0 + j) * K8_KEYS + c, seen.count - 1));
                const int page = (int)min((unsigned)entry, (unsigned)(a.pages - 1));
                return ((uint32_t)page * 2 * a.nkv + kvh) * a.page.size + (uint32_t)(key - page_of(a.page, key) * a.page.size);
            };
            auto keep = [&](int j, int c, uint32_t row, int kb, int vb) {
                const int at = (j & 7) * 128 + c;
                const bool bad = kb == KV8_BAD_BYTE || vb == KV8_BAD_BYTE;
                row_s[at] = row;
                kf_s[at] = bad ? __int_as_float(0x7fc00000) : kv8_scale(kb);
                vf_s[at] = kv8_value_factors(bad ? 0 : vb - 127);
            };
            const bool two = kt < 32;
            // table entries are read two tiles ahead of their rows' use, scales one (a warp issues in order, and would
            // stand still at the first use of what it just asked for)
            int ea = 0, eb = 0, ka = 0, va = 0, kb = 0, vb = 0;
            uint32_t ra = 0, rb = 0;
            auto ask_rows = [&](int j) {
                if (j >= ntiles) return;
                ra = row_of(j, kt, ea);
                ka = a.scales[ra];
                va = a.scales[ra + plane];
                if (two) {
                    rb = row_of(j, kt + 96, eb);
                    kb = a.scales[rb];
                    vb = a.scales[rb + plane];
                }
            };
            auto ask_entries = [&](int j) {
                if (j >= ntiles) return;
                ea = entry_of(j, kt);
                if (two) eb = entry_of(j, kt + 96);
            };
            auto tell = [&](int j) {
                if (j >= ntiles) return;
                keep(j, kt, ra, ka, va);
                if (two) keep(j, kt + 96, rb, kb, vb);
                mbar_arrive(rows_full + 8 * (j & 7));
            };
            ask_entries(0);
            ask_rows(0);
            ask_entries(1);
#pragma unroll 1
            for (int j = 0; j < AHEAD; ++j) {
                tell(j);
                ask_rows(j + 1);
                ask_entries(j + 2);
            }
            bool ok = true;
            for (int j = 0; j < ntiles && ok; ++j) {
                const int s = j & 1;
                tell(j + AHEAD);
                ask_rows(j + AHEAD + 1);
                ask_entries(j + AHEAD + 2);
                // the tile's place is free when the scores of the tile before the last are done
                if (!pt_wait_warp(rows_full + 8 * (j & 7), ((uint32_t)j >> 3) & 1u) ||
                    !pt_wait_warp(k_empty + 8 * s, (((uint32_t)j >> 1) & 1u) ^ 1u)) {
                    if (lane == 0) atomicExch(a.error_word, 33);
                    ok = false;
                    break;
                }
                const uint32_t tile = tc_smem(k_s + s * KT);
                constexpr int N = (128 * CPR + 95) / 96;
                uint32_t rows[N];
#pragma unroll
                for (int i = 0; i < N; ++i) rows[i] = row_s[(j & 7) * 128 + min(kt + i * 96, 128 * CPR - 1) / CPR];
#pragma unroll
                for (int i = 0; i < N; ++i) {
                    const int at = kt + i * 96;
                    if (at < 128 * CPR)
                        cp_async_16(tile + k8_code_place<HD>(at / CPR, at % CPR), a.codes + (size_t)rows[i] * HD + at % CPR * 16, 16);
                }
                cp_async_commit();
                if (j > 0) {
                    cp_async_wait<1>();
                    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                    mbar_arrive(k_full + 8 * (s ^ 1));
                }
                if (j + 1 == ntiles) {
                    cp_async_wait<0>();
                    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                    mbar_arrive(k_full + 8 * s);
                }
            }
            cp_async_wait<0>();
        } else if (ntiles > 0) {
            // ------------------------------------------------------------------ the products
            constexpr uint32_t idesc_s = k8_idesc_codes(K8_ROWS, K8_KEYS), idesc_o = pt_idesc(K8_ROWS, HD, 1);
            const uint32_t leader = k8_elect();
            // low words: the address in units of 16 bytes (below 2^14 of them), the leading byte offset from bit 16 on
            const uint32_t q_low = tc_smem(q_s) >> 4 | 1u << 16, k_low = tc_smem(k_s) >> 4 | 1u << 16;
            const uint32_t v_low = tc_smem(v_s) >> 4 | (uint32_t)(K8_KEYS * 128 >> 4) << 16;
            // row tile x with the keys of tile j; its weights with the values of tile j, `first` of its tiles
            auto scores = [&](int x, int j) {
                const uint32_t qa = q_low + (PAIR ? 0u : (uint32_t)(x * 2 * QT >> 4)), ka = k_low + (uint32_t)((j & 1) * KT >> 4);
#pragma unroll
                for (int part = 0; part < 2; ++part)
#pragma unroll
                    for (int kk = 0; kk < HD / 32; ++kk)
                        k8_mma_codes(leader, tmem + x * 128, qa + (uint32_t)((part * QT + kk * 32) >> 4),
                                     ka + (uint32_t)(kk * 32 >> 4), k8_codes_high<HD>(), idesc_s, (part | kk) != 0);
                k8_commit(leader, s_full + 8 * x);
            };
            auto output = [&](int x, int j, bool first) {
                const uint32_t va = v_low + (uint32_t)((j & 1) * VT >> 4);
#pragma unroll
                for (int kk = 0; kk < K8_KEYS / 16; ++kk)
                    k8_mma_weights(leader, tmem + 256 + x * HD, tmem + x * 128 + kk * 8, va + (uint32_t)(kk * 16 * 128 >> 4),
                                   k8_values_high(), idesc_o, !first || kk != 0);
            };
            bool ok = pt_wait_warp(q_ready, 0) && (PAIR || !has_b || pt_wait_warp(q_ready + 8, 0)) && pt_wait_warp(k_full, 0);
            // a product that overwrites weights follows the one that reads them: one warp's products run in their order
            if constexpr (PAIR) {
                // tile j: row tile j & 1
                if (ok) {
                    pt_fence_after();
                    scores(0, 0);
                    k8_commit(leader, k_empty);
                    if (ntiles > 1) {
                        ok = pt_wait_warp(k_full + 8, 0);
                        pt_fence_after();
                        if (ok) {
                            scores(1, 1);
                            k8_commit(leader, k_empty + 8);
                        }
                    }
                }
                for (int j = 0; j < ntiles && ok; ++j) {
                    const int s = j & 1;
                    const uint32_t ph = ((uint32_t)j >> 1) & 1u;
                    ok = pt_wait_warp(v_full + 8 * s, ph) && pt_wait_warp(p_ready + 8 * s, ph);
                    if (!ok) break;
                    pt_fence_after();
                    output(s, j, j < 2);
                    k8_commit(leader, v_empty + 8 * s);
                    if (j + 2 < ntiles) {
                        ok = pt_wait_warp(k_full + 8 * s, ph ^ 1u);
                        if (!ok) break;
                        pt_fence_after();
                        scores(s, j + 2);
                        k8_commit(leader, k_empty + 8 * s);
                    } else {
                        k8_commit(leader, o_full + 8 * s);
                    }
                }
            } else {
                if (ok) {
                    pt_fence_after();
                    scores(0, 0);
                    if (has_b) scores(1, 0);
                    k8_commit(leader, k_empty);
                }
                for (int j = 0; j < ntiles && ok; ++j) {
                    const uint32_t ph = ((uint32_t)j >> 1) & 1u, ph1 = ((uint32_t)(j + 1) >> 1) & 1u;
                    const int s = j & 1, s1 = s ^ 1;
                    const bool more = j + 1 < ntiles;
                    ok = pt_wait_warp(v_full + 8 * s, ph) && pt_wait_warp(p_ready, (uint32_t)j & 1u);
                    if (!ok) break;
                    pt_fence_after();
                    output(0, j, j == 0);
                    if (!has_b) k8_commit(leader, v_empty + 8 * s);
                    if (more) {
                        ok = pt_wait_warp(k_full + 8 * s1, ph1);
                        if (!ok) break;
                        pt_fence_after();
                        scores(0, j + 1);
                        if (!has_b) k8_commit(leader, k_empty + 8 * s1);
                    } else {
                        k8_commit(leader, o_full);
                    }
                    if (has_b) {
                        ok = pt_wait_warp(p_ready + 8, (uint32_t)j & 1u);
                        if (!ok) break;
                        pt_fence_after();
                        output(1, j, j == 0);
                        k8_commit(leader, v_empty + 8 * s);
                        if (more) {
                            scores(1, j + 1);
                            k8_commit(leader, k_empty + 8 * s1);
                        } else {
                            k8_commit(leader, o_full + 8);
                        }
                    }
                }
            }
            if (!ok && lane == 0) atomicExch(a.error_word, 32);
        }
    } else if (warp >= 8) {
        // ---------------------------------------------------------------------- values
        k8_less_registers<80>();
        constexpr int NP = CPR;                              // passes
        // eight neighbouring lanes: two rows' four runs, whose stores then fall into different banks
        const int run = HD == 128 ? (lane & 3) | ((lane >> 1) & 4) : lane & 3;
        const int sub = HD == 128 ? ((lane >> 2) & 1) | ((lane >> 3) & 2) : lane >> 2;
        const int r0 = (warp - 8) * (RP / 4) + sub;
        auto load_values = [&](int j, uint4 (&x)[NP]) {
#pragma unroll
            for (int i = 0; i < NP; ++i)
                x[i] = *reinterpret_cast<const uint4*>(
                    a.codes + ((size_t)row_s[(j & 7) * 128 + i * RP + r0] + plane) * HD + run * 16);
        };
        // PAIR: a thread's runs lie in shared memory from their copy to their use, read by itself alone
        const int vt = (warp - 8) * 32 + lane;
        auto copy_values = [&](int j) {
            if (j < ntiles) {
#pragma unroll
                for (int i = 0; i < NP; ++i)
                    cp_async_16(tc_smem(raw_s + (j % K8_AHEAD * NP + i) * 128 + vt),
                                a.codes + ((size_t)row_s[(j & 7) * 128 + i * RP + r0] + plane) * HD + run * 16, 16);
            }
            cp_async_commit();
        };
        auto store_values = [&](int j, const uint4 (&x)[NP]) {
#pragma unroll
            for (int i = 0; i < NP; ++i) {
                const int r = i * RP + r0, c = run * 2;
                const uint32_t f = vf_s[(j & 7) * 128 + r], f1 = __byte_perm(f, f, 0x1010);
                const uint32_t in[4] = {x[i].x, x[i].y, x[i].z, x[i].w};
                uint32_t out[8];
#pragma unroll
                for (int k = 0; k < 4; ++k) {       // codes 0 and 2 of a word, then 1 and 3
                    out[2 * k] = kv8_mul_bf16x2(((in[k] << 8) & 0x80008000u) | ((in[k] << 4) & 0x07f007f0u), f1);
                    out[2 * k + 1] = kv8_mul_bf16x2((in[k] & 0x80008000u) | ((in[k] >> 4) & 0x07f007f0u), f1);
                }
                if ((f >> 16) != 0x3f80u) {         // values above 2^15
                    const uint32_t f2 = __byte_perm(f, f, 0x3232);
#pragma unroll
                    for (int k = 0; k < 8; ++k) out[k] = kv8_mul_bf16x2(out[k], f2);
                }
                unsigned char* base = v_s + (j & 1) * VT + (c >> 3) * (128 * 128) + r * 128;
                *reinterpret_cast<uint4*>(base + (((c & 7) ^ (r & 7)) << 4)) = make_uint4(out[0], out[1], out[2], out[3]);
                *reinterpret_cast<uint4*>(base + ((((c & 7) + 1) ^ (r & 7)) << 4)) = make_uint4(out[4], out[5], out[6], out[7]);
            }
        };
        if (ntiles > 0) {
            uint4 vx[NP];
            bool ok = true;
            auto rows_there = [&](int j) { return pt_wait_warp(rows_full + 8 * (j & 7), ((uint32_t)j >> 3) & 1u); };
            if constexpr (PAIR) {
                for (int j = 0; j < AHEAD && ok; ++j) {
                    ok = j >= ntiles || rows_there(j);
                    if (ok) copy_values(j);
                }
            } else {
                ok = rows_there(0);
                if (ok) load_values(0, vx);
            }
            for (int j = 0; j < ntiles && ok; ++j) {
                const int s = j & 1;
                if constexpr (PAIR) {
                    cp_async_wait<K8_AHEAD - 1>();
#pragma unroll
                    for (int i = 0; i < NP; ++i) vx[i] = raw_s[(j % K8_AHEAD * NP + i) * 128 + vt];
                }
                ok = pt_wait_warp(v_empty + 8 * s, (((uint32_t)j >> 1) & 1u) ^ 1u);
                if (!ok) break;
                store_values(j, vx);
                asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                mbar_arrive(v_full + 8 * s);
                if constexpr (PAIR) {
                    ok = j + AHEAD >= ntiles || rows_there(j + AHEAD);
                    if (ok) copy_values(j + AHEAD);
                } else if (j + 1 < ntiles) {
                    ok = rows_there(j + 1);
                    if (ok) load_values(j + 1, vx);
                }
            }
            if constexpr (PAIR) cp_async_wait<0>();
            if (!ok && lane == 0) atomicExch(a.error_word, 34);
        }
    } else {
        // ------------------------------------------------------------------------- softmax, a row a thread
        k8_more_registers<184>();
        const int x = warp >> 2, r = tid & 127;
        const int tok = tok0 + (PAIR ? 0 : x * TPT) + min(r, RPT - 1) / G;
        const bool valid = r < RPT && tok < q_len;
        const size_t head = (size_t)(q_start + min(tok, q_len - 1)) * a.nq + kvh * G + r % G;
        const uint32_t lanes = (uint32_t)((warp & 3) * 32) << 16;
        const uint32_t t_s = tmem + lanes + x * 128, t_o = tmem + lanes + 256 + x * HD;
        float m = -INFINITY, l = 0.f, row_scale = 0.f;
        bool ok = true;
        if (x == 0 || has_b) {
            if (ntiles > 0) {
                // The query: two codes a number, into the K-major swizzled tiles.  A warp's 32 rows, the lanes side by side on
                // a row (a lane on a row of its own reads 32 lines with every load: 12,000 clocks instead of 6,000, most of
                // which are conversions).
                constexpr int LR = HD / 8, RI = 32 / LR;          // lanes of a row, rows of a load
                const uint32_t from = valid ? (uint32_t)(((size_t)(q_start + tok) * a.q_stride + (size_t)(kvh * G + r % G) * HD) >> 3)
                                            : 0xffffffffu;
                int byte = 0;
#pragma unroll 1
                for (int i0 = 0; i0 < 32 / RI; i0 += 8) {
                    uint4 in[8];
#pragma unroll
                    for (int i = 0; i < 8; ++i) {
                        const uint32_t at = __shfl_sync(0xffffffffu, from, (i0 + i) * RI + lane / LR);
                        in[i] = make_uint4(0u, 0u, 0u, 0u);
                        if (at != 0xffffffffu) in[i] = *reinterpret_cast<const uint4*>(a.q + ((size_t)at << 3) + lane % LR * 8);
                    }
#pragma unroll
                    for (int i = 0; i < 8; ++i) {
                        uint32_t w[4] = {in[i].x, in[i].y, in[i].z, in[i].w}, most = 0u, hi[2], lo[2];
#pragma unroll
                        for (int k = 0; k < 4; ++k) most = __vmaxu2(most, w[k] & 0x7fff7fffu);
#pragma unroll
                        for (int o = LR / 2; o > 0; o >>= 1) most = __vmaxu2(most, __shfl_xor_sync(0xffffffffu, most, o));
                        const int b8 = kv8_scale_byte(__uint_as_float(max(most << 16, most & 0xffff0000u)));
                        const uint32_t keep = b8 != KV8_BAD_BYTE ? 0xffffffffu : 0u;      // a query that is not finite gives NaNs
                        const uint32_t inv = __float_as_uint(kv8_inverse_scale(b8 & 0xff & (int)keep));
#pragma unroll
                        for (int k = 0; k < 4; ++k) {             // two numbers, exact as float16 (below 2^-14 in value: nearly)
                            w[k] &= keep;
                            const uint64_t v = k8_mul2(k8_two(w[k] << 16, w[k] & 0xffff0000u), k8_two(inv, inv));
                            const __half2 x2 = __floats2half2_rn(k8_lo(v), k8_hi(v));
                            const uint32_t c = __nv_cvt_halfraw2_to_fp8x2(x2, __NV_SATFINITE, __NV_E4M3);
                            const __half2 b2 = __nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)c, __NV_E4M3);
                            const uint32_t d = __nv_cvt_halfraw2_to_fp8x2(__hsub2(x2, b2), __NV_SATFINITE, __NV_E4M3);
                            hi[k >> 1] = (k & 1) ? hi[k >> 1] | c << 16 : c;
                            lo[k >> 1] = (k & 1) ? lo[k >> 1] | d << 16 : d;
                        }
                        const int mine = __shfl_sync(0xffffffffu, b8, lane % RI * LR);
                        if (lane / RI == i0 + i) byte = mine;
                        if (PAIR && x == 1) continue;             // (the same rows as x = 0)
                        unsigned char* to = q_s + x * 2 * QT + (lane & 1) * 8 +
                                            k8_code_place<HD>((r & ~31) + (i0 + i) * RI + lane / LR, lane % LR >> 1);
                        *reinterpret_cast<uint2*>(to) = make_uint2(hi[0], hi[1]);
                        *reinterpret_cast<uint2*>(to + QT) = make_uint2(lo[0], lo[1]);
                    }
                }
                // (never zero, however small the scale: a score that is not seen is -inf before the product)
                row_scale = byte != KV8_BAD_BYTE ? fmaxf(kv8_scale(byte) * a.scale_log2e, 1.17549435e-38f) : __int_as_float(0x7fc00000);
                asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                if (!PAIR || x == 0) mbar_arrive(q_ready + 8 * x);
            }
            // in counts of seen keys: the newest key of this row and the newest one that its window has passed
            const int pos = past + min(tok, q_len - 1), shift = seen.kept - seen.lo;
            const int v_max = pos + shift, v_min = a.window > 0 ? pos - a.window + shift : -1;
            // of the tile's rows: the least v_max, the largest v_min
            const int first_tok = tok0 + (PAIR ? 0 : x * TPT);
            const int all_max = past + first_tok + shift;
            const int all_min = a.window > 0 ? past + min(first_tok + TPT, q_len) - 1 - a.window + shift : -1;
            constexpr int STEP = PAIR ? 2 : 1;
            for (int j = PAIR ? x : 0; j < ntiles; j += STEP) {
                if (!pt_wait_warp(s_full + 8 * x, (uint32_t)(j / STEP) & 1u)) {
                    if (lane == 0) atomicExch(a.error_word, 35);
                    ok = false;
                    break;
                }
                pt_fence_after();
                const float4* kf = reinterpret_cast<const float4*>(kf_s + (j & 7) * 128);
                const int v0 = (tile0 + j) * K8_KEYS;
                uint64_t t[64];                         // scores times their key's scale, in pairs
                {
                    uint32_t s[2][32];
                    pt_ld32(t_s, s[0]);
#pragma unroll
                    for (int c = 0; c < 4; ++c) {
                        pt_wait_ld();
                        if (c < 3) pt_ld32(t_s + (c + 1) * 32, s[(c + 1) & 1]);
                        const uint32_t* sc = s[c & 1];
#pragma unroll
                        for (int i = 0; i < 32; i += 4) {
                            const float4 f = kf[c * 8 + (i >> 2)];
                            t[c * 16 + (i >> 1)] = k8_mul2(k8_two(sc[i], sc[i + 1]),
                                                           k8_two(__float_as_uint(f.x), __float_as_uint(f.y)));
                            t[c * 16 + (i >> 1) + 1] = k8_mul2(k8_two(sc[i + 2], sc[i + 3]),
                                                               k8_two(__float_as_uint(f.z), __float_as_uint(f.w)));
                        }
                    }
                }
                if (v0 + K8_KEYS - 1 > all_max || v0 <= all_min) {
#pragma unroll
                    for (int c = 0; c < 4; ++c) {
                        const int b = v0 + c * 32;
                        const uint32_t seen_bits = k8_below(v_max + 1 - b) & ~(k8_below(v_min + 1 - b) & ~k8_below(a.keep_first - b));
#pragma unroll
                        for (int i = 0; i < 16; ++i) {
                            uint32_t lo = (uint32_t)t[c * 16 + i], hi = (uint32_t)(t[c * 16 + i] >> 32);
                            if (!(seen_bits >> (2 * i) & 1u)) lo = 0xff800000u;          // -inf
                            if (!(seen_bits >> (2 * i + 1) & 1u)) hi = 0xff800000u;
                            t[c * 16 + i] = k8_two(lo, hi);
                        }
                    }
                }
                float mx[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
                for (int i = 0; i < 16; ++i)
#pragma unroll
                    for (int c = 0; c < 4; ++c) mx[c] = fmaxf(fmaxf(mx[c], k8_lo(t[c * 16 + i])), k8_hi(t[c * 16 + i]));
                const float top = fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3])) * row_scale;
                float alpha = 1.f;
                if (top > m + K8_SLACK) {
                    alpha = pt_ex2(m - top);
                    m = top;
                }
                // a row that has seen nothing yet: weights of exp(-inf) whatever finite number is taken off
                const float ref = m == -INFINITY ? 0.f : m;
                const uint64_t ref2 = k8_two(__float_as_uint(-ref), __float_as_uint(-ref));
                const uint64_t scale2 = k8_two(__float_as_uint(row_scale), __float_as_uint(row_scale));
                l *= alpha;
                uint64_t sum[2] = {0ull, 0ull};
                uint32_t packed[2][32];
#pragma unroll
                for (int i = 0; i < 64; ++i) {
                    const uint64_t d = k8_fma2(t[i], scale2, ref2);
                    const float p0 = pt_ex2(k8_lo(d)), p1 = pt_ex2(k8_hi(d));
                    sum[i & 1] = k8_add2(sum[i & 1], k8_two(__float_as_uint(p0), __float_as_uint(p1)));
                    packed[i >> 5][i & 31] = pack_bf16(p0, p1);
                }
                const uint64_t both = k8_add2(sum[0], sum[1]);
                l += k8_lo(both) + k8_hi(both);
                if (j >= STEP && __any_sync(0xffffffffu, alpha != 1.f)) {
                    // (the scores came after the product before on the tensor cores: the output is at rest)
#pragma unroll 1
                    for (int c0 = 0; c0 < HD; c0 += 32) {
                        uint32_t o[32];
                        pt_ld32(t_o + c0, o);
                        pt_wait_ld();
#pragma unroll
                        for (int i = 0; i < 32; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * alpha);
                        pt_st32(t_o + c0, o);
                    }
                }
                pt_st32(t_s, packed[0]);
                pt_st32(t_s + 32, packed[1]);
                pt_wait_st();
                pt_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(p_ready + 8 * x);
            }
            const bool some = PAIR ? ntiles > x : ntiles > 0;         // whether there is an output
            if (some && ok && !pt_wait_warp(o_full + 8 * x, 0)) {
                if (lane == 0) atomicExch(a.error_word, 36);
                ok = false;
            }
            pt_fence_after();
            // ---------------------------------------------------------------- epilogue
            if (ok) {
                const bool parts = PAIR || splits > 1, stored = valid && (!parts || kv8_has_room(a.parts, (int)(head / a.nq)));
                // (head h's part is part0 + h * splits; modulo 2^64 where the difference is negative)
                const size_t part0 = (size_t)(PAIR ? 2 * split + x : split) -
                                     (parts ? (size_t)kv8_first_token(a.parts) * a.nq * a.parts.splits : 0);
                const size_t at = part0 + head * a.parts.splits;
                const float f = parts ? 1.f : l == 0.f ? 0.f : 1.f / l;
                if (parts && stored) {
                    a.parts.ml[2 * at] = l == 0.f ? -INFINITY : m;
                    a.parts.ml[2 * at + 1] = l;
                }
                // A row's pieces of 128 bytes go through shared memory, a warp's 32 rows by themselves, and are stored by eight
                // lanes each (a lane storing its own row touches 32 lines with every store: 6,000 clocks instead of 4,000).
                unsigned char* piece = out_s + (warp * 32 + lane) * 128;
                const uint32_t to = stored ? (uint32_t)head : 0xffffffffu;
                const int pieces = parts ? HD / 32 : HD / 64;
#pragma unroll 1
                for (int c = 0; c < pieces && (some || !parts); ++c) {
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        uint32_t o[32];
                        if (h == 1 && parts) break;
                        const int c0 = parts ? c * 32 : c * 64 + h * 32;
                        if (some) {
                            pt_ld32(t_o + c0, o);
                            pt_wait_ld();
                        } else {                                   // rows that see nothing at all
#pragma unroll
                            for (int i = 0; i < 32; ++i) o[i] = 0u;
                        }
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            float v[8];
#pragma unroll
                            for (int k = 0; k < 8; ++k)            // (places 1 and 2 of four hold features 2 and 1)
                                v[k] = __uint_as_float(o[8 * i + ((k & 3) == 1 ? k + 1 : (k & 3) == 2 ? k - 1 : k)]) * f;
                            if (parts) {
                                *reinterpret_cast<float4*>(piece + ((2 * i ^ (lane & 7)) << 4)) = make_float4(v[0], v[1], v[2], v[3]);
                                *reinterpret_cast<float4*>(piece + (((2 * i + 1) ^ (lane & 7)) << 4)) = make_float4(v[4], v[5], v[6], v[7]);
                            } else {
                                store8(reinterpret_cast<bf16*>(piece + (((4 * h + i) ^ (lane & 7)) << 4)), v);
                            }
                        }
                    }
                    __syncwarp();
#pragma unroll
                    for (int i = 0; i < 8; ++i) {
                        const int rr = i * 4 + (lane >> 3);
                        const uint32_t h = __shfl_sync(0xffffffffu, to, rr);
                        const uint4 v = *reinterpret_cast<const uint4*>(out_s + (warp * 32 + rr) * 128 + (((lane & 7) ^ (rr & 7)) << 4));
                        if (h != 0xffffffffu) {
                            if (parts)
                                *reinterpret_cast<uint4*>(a.parts.o + (part0 + (size_t)h * a.parts.splits) * HD + c * 32 + (lane & 7) * 4) = v;
                            else
                                *reinterpret_cast<uint4*>(a.out + (size_t)h * HD + c * 64 + (lane & 7) * 8) = v;
                        }
                    }
                    __syncwarp();
                }
            }
        }
    }
    pt_fence_before();
    __syncthreads();
    pdl_launch_dependents();
    if (warp == 12) {
        pt_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512u) : "memory");
    }
}

template <int HD, bool PAIR> static int launch_kv8_tc(const Kv8TcArgs& a, dim3 grid, cudaStream_t s) {
    auto kernel = kv8_attention_tc_kernel<HD, PAIR>;
    // more than half of an SM's shared memory, so that no second CTA lands there and waits for tensor memory
    const int smem = k8_smem(HD, PAIR) > 120 * 1024 ? k8_smem(HD, PAIR) : 120 * 1024;
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
    e = mstar_launch(kernel, grid, dim3(K8_THREADS), (size_t)smem, s, a);
    return e != cudaSuccess ? (int)e : launch_status();
}

// Entries [first_entry, first_entry + count) of at most max_q tokens each.  q rows q_stride apart, 16-byte aligned.
// `tokens`, `splits`, `part_o` and `part_ml` as in mstar_kv8_attention; `pair`: max_q is at most 128 / G, and a CTA takes
// the even and the odd key tiles of its one row tile side by side and leaves two of the (an even number of) parts.  Returns 0, a CUDA error code or -1 (shape
// refused).
MSTAR_API int mstar_kv8_attention_tc(const void* q, int q_stride, void* out, const void* codes, const void* scales, int pages,
                                     const int* block_table, int bt_stride, int bt_width, const int* qo_indptr, const int* kv_len,
                                     int first_entry, int count, int max_q, int tokens, int nq, int nkv, int hd,
                                     int page_size, int window, int keep_first, float scale, int splits, int pair,
                                     float* part_o, float* part_ml, int* error_word, void* stream) {
    if (count <= 0 || max_q <= 0) return 0;
    if ((hd != 64 && hd != 128) || nkv <= 0 || nq % nkv != 0 || nq / nkv > K8_ROWS || page_size <= 0 ||
        pages <= 0 || bt_width <= 0 || splits < 1 || count > 65535 || error_word == nullptr || !(scale > 0.f) || ((uintptr_t)q & 15) != 0 ||
        q_stride % 8 != 0 || ((uintptr_t)codes & 15) != 0 || ((uintptr_t)out & 15) != 0 ||
        (long long)pages * 2 * nkv * page_size > 0xffffffffll)
        return -1;
    const Kv8Parts parts{part_o, part_ml, splits, qo_indptr + first_entry, count, tokens};
    const Kv8TcArgs a{(const bf16*)q, (bf16*)out, (const uint8_t*)codes, (const uint8_t*)scales, block_table, qo_indptr,
                      kv_len, q_stride, bt_stride, bt_width, pages, nq, nkv, window, keep_first, first_entry,
                      scale * 1.4426950408889634f, page_split(page_size), parts, error_word};
    const int per_tile = K8_ROWS / (nq / nkv);
    if (pair && (max_q > per_tile || splits % 2 != 0)) return -1;
    const long long tiles = pair ? 1 : ((long long)max_q + 2 * per_tile - 1) / (2 * per_tile);
    if (tiles > 65535) return -1;
    const dim3 grid(nkv * (pair ? splits / 2 : splits), (unsigned)tiles, count);
    const cudaStream_t s = (cudaStream_t)stream;
    int code;
    if (pair) code = hd == 64 ? launch_kv8_tc<64, true>(a, grid, s) : launch_kv8_tc<128, true>(a, grid, s);
    else code = hd == 64 ? launch_kv8_tc<64, false>(a, grid, s) : launch_kv8_tc<128, false>(a, grid, s);
    if (code != 0 || splits == 1) return code;
    return kv8_merge(parts, out, MSTAR_BF16, nq, hd, s);
}

MSTAR_API int mstar_kv8_attention_tc_packed(const long long* a) {
    return mstar_kv8_attention_tc((const void*)a[0], (int)a[1], (void*)a[2], (const void*)a[3], (const void*)a[4],
        (int)a[5], (const int*)a[6], (int)a[7], (int)a[8], (const int*)a[9], (const int*)a[10], (int)a[11], (int)a[12],
        (int)a[13], (int)a[14], (int)a[15], (int)a[16], (int)a[17], (int)a[18], (int)a[19], (int)a[20],
        kv8_packed_float(a[21]), (int)a[22], (int)a[23], (float*)a[24], (float*)a[25], (int*)a[26], (void*)a[27]);
}
