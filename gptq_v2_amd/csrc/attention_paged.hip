// Attention of a few query tokens per sequence over a paged cache of 8-bit keys and values (the layout and the scales
// that kv_append.hip writes): a decoder's step for one new token, or for the several of a checked draft or a chunk.
//
// With K = ks[page] k8 and V = vs[page] v8, in powers of two (c = softmax scale * log2 e), and any whole number e per page:
//   y_t = c ks (q . k8_t) + log2 vs - e,  w_t = 2^(y_t - M + 7),  O = sum_t w_t (2^e v8_t) / sum_t w_t 2^e / vs
// for a reference M near max y.  2^e v8 is exact in fp16 for e from -15 (the smallest code is 2^-9) to 7 (the largest 448),
// and costs nothing: the conversion of codes takes a factor.  So e is the scale's own exponent less that of the first page the
// wave sees, as far as that range goes: within it w_t is the softmax weight alone and small scales cost it nothing; what lies
// outside stays in the exponent y, and the denominator takes it out again in 32 bits.
// The weights meet the codes on the matrix core in fp16, rounded once (11 bits, against 8 in bf16); the denominator sums them
// unrounded.  fp16 has 11 bits down to 2^-14 and steps of 2^-24 below.  M lags up to 8 behind the maximum (see there), so the
// largest weight of a row is 2^7 to 2^15 (of 65504): a weight keeps its bits down to 2^-21 of it, and what is lost below is
// 2^-32 of it.
//
// A wave takes 64 tokens at a time: S^T = K Q^T (16 x 16 x 32 tiles: tokens by query rows) and O^T = V^T P^T.  Row
// 4 g + i of the S^T tile a stands for token 16 g + 4 a + i; lane group g then holds, as the tiles' results, the weights of
// the 16 adjacent tokens 16 g .. 16 g + 15 of its query row -- exactly what it has to supply as the operand P^T, next to
// the 16 bytes of a row of V^T.  No value crosses lanes but for the maximum.
// The codes come through LDS: the matrix operands want 16 lanes in 16 different rows, and loads of 16 bytes each from 16
// rows reach 4.7 TB/s where the same bytes in order reach 6.  The asynchronous copy brings whole lines, its 16-byte
// pieces permuted within 128 so that the operand reads touch all banks.  A wave has its own buffers and waits for
// nobody: the next tile's keys are under way as soon as this one's have met the queries, its values after this one's
// have met the weights.
// The rows are the query heads that share a kv head (times the tokens of the sequence); the cache is read once for
// every 16 NQ of them.  e4m3 codes are exact in either 16-bit type: Q K^T runs in q's type.
//
// Bound by HBM: 2 head_dim bytes per cached token and kv head.  A long sequence is cut into runs of tokens for several
// workgroups, whose (O, M, l) a second kernel joins.
// Measured at 64 heads on 8, 128 channels, pages of 64, on operands that no cache holds: one token each of 64 sequences of 391
// to 8192 131 us (5.0 TB/s), of 128 sequences of 2048 98 us (5.5 TB/s); four tokens of one sequence of 131071 73.5 us (3.65
// TB/s, the join 5.5 us of it: the copies alone take 43 us, and the decoding, products and exponentials of 32 query rows hide
// behind them only in part); 100 tokens of 32 heads 5.9 us (a launch).  On cached operands 512 tokens behind 7680 200 us (667 TFLOP/s).
#include <type_traits>

#include "gq_common.h"

namespace {

constexpr int PA_MAX_SPLITS = 64;   // one wave weighs them
constexpr int PA_MAX_LEN = 1 << 30;     // longest sequence; tables are narrower (a longer one is NaN)
constexpr int PA_NO_EXPONENT = 1000;
constexpr float PA_LOG2E = 1.44269504088896340736f;

struct PagedArgs {
    const void *q;
    void *out;
    int64_t q_tok, q_head, o_tok, o_head;   // strides in elements
    const uint8_t *k_codes, *v_codes;
    const float *k_scale, *v_scale;
    const int32_t *table, *lens, *cu;       // cu NULL: one query token per sequence
    float *part_o, *part_ml;                // partial results: [token][head][split][head_dim], [token][head][split][2]
    int64_t n_tokens;
    int n_pages, table_width;
    int batch, n_heads, n_kv_heads, group, head_dim, page_log2, tiles_per_split, n_splits, n_items;
    float scale;                            // softmax scale * log2 e
};

// A uniform load of what no kernel writes meanwhile, by the scalar unit: it is not counted with the copies, whose
// order the waits below rely on.
template <typename V>
__device__ __forceinline__ V pa_scalar_load(const V *p, int64_t i)
{
    return *(const V __attribute__((address_space(4))) *)(uintptr_t)(p + i);
}

__device__ __forceinline__ int pa_exponent(float x) { return (int)(__float_as_uint(x) >> 23 & 0xff) - 127; }

// At most N of the wave's copies are left under way; the oldest end first.
template <int N>
__device__ __forceinline__ void pa_wait()
{
    static_assert(N == 0 || N == 4 || N == 8, "");
    if constexpr (N == 8) asm volatile("s_waitcnt vmcnt(8)" ::: "memory");
    else if constexpr (N == 4) asm volatile("s_waitcnt vmcnt(4)" ::: "memory");
    else asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __builtin_amdgcn_sched_barrier(0);
}

// The wave's reads of a buffer have returned: a copy may overwrite it.
__device__ __forceinline__ void pa_reads_done()
{
    __builtin_amdgcn_sched_barrier(0);
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    __builtin_amdgcn_sched_barrier(0);
}

template <typename T> struct Mfma;
template <> struct Mfma<_Float16> {
    typedef f16x8 vec;
    static __device__ __forceinline__ f32x4 run(f16x8 a, f16x8 b, f32x4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0); }
    // 8 codes (two words) times a power of two from 2^-15 to 2^7 to the operand's type, exactly
    static __device__ __forceinline__ f16x8 decode(unsigned lo, unsigned hi, float f = 1.f)
    {
        const f16x2 a = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(lo, f, false), b = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(lo, f, true);
        const f16x2 c = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(hi, f, false), d = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(hi, f, true);
        return f16x8{a[0], a[1], b[0], b[1], c[0], c[1], d[0], d[1]};
    }
};
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
template <> struct Mfma<__bf16> {
    typedef bf16x8 vec;
    static __device__ __forceinline__ f32x4 run(bf16x8 a, bf16x8 b, f32x4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0); }
    static __device__ __forceinline__ bf16x8 decode(unsigned lo, unsigned hi)
    {
        const bf16x2 a = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, 1.f, false), b = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, 1.f, true);
        const bf16x2 c = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, 1.f, false), d = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, 1.f, true);
        return bf16x8{a[0], a[1], b[0], b[1], c[0], c[1], d[0], d[1]};
    }
};

// Sequence, first row and token rows of a workgroup's item.  With cu, sequence b's row tiles start at item
// cu[b] group / MR + b, which leaves each sequence room for all its tiles without the host knowing the lengths.
struct Item {
    int b, tile;
    int64_t row0;   // first query token's row in q
    int n;          // query tokens of the sequence; 0: nothing to do
    int len;        // its cached tokens
};

__device__ __forceinline__ Item find_item(const PagedArgs &a, int item, int mr)
{
    if (!a.cu) {
        const int tiles = (a.group + mr - 1) / mr;
        const int b = item / tiles;
        return {b, item - b * tiles, b, 1, a.lens[b]};
    }
    // The starts rise: the item's sequence is the last of those that start at or before it; 64 are looked at at a time, and
    // what is wanted of it is nearly always in the lanes.
    const int lane = threadIdx.x & 63;
    int lo = -1, c = 0, mine = 0, len = 0;
    for (int b0 = 0; b0 < a.batch; b0 += 64) {
        const int at = b0 + lane < a.batch ? b0 + lane : a.batch;
        mine = a.cu[at];
        len = a.lens[at < a.batch ? at : a.batch - 1];
        c = __popcll(__ballot(b0 + lane < a.batch && (int64_t)mine * a.group / mr + at <= item));
        lo += c;
        if (c < 64) break;
    }
    if (lo < 0) return {0, 0, 0, 0, 0};
    lo = __builtin_amdgcn_readfirstlane(lo);
    c = __builtin_amdgcn_readfirstlane(c);
    const bool here = c > 0 && c < 64;
    const int64_t row0 = here ? __builtin_amdgcn_readlane(mine, c - 1) : a.cu[lo];
    const int64_t n = (here ? __builtin_amdgcn_readlane(mine, c) : a.cu[lo + 1]) - row0, tile = item - (row0 * a.group / mr + lo);
    if (row0 < 0 || n <= 0 || row0 + n > a.n_tokens || tile < 0 || tile * mr >= n * a.group) return {lo, 0, 0, 0, 0};
    return {lo, (int)tile, row0, (int)n, here ? (int)__builtin_amdgcn_readlane(len, c - 1) : a.lens[lo]};
}

// Piece p (of 16 bytes) of the 128 bytes R of a buffer lies in place p ^ swizzle(R).  16 lanes read 16 pieces at a time
// over 256 bytes of banks: of 16 adjacent channels' values, of the keys of tokens 16 b + 4 i + 0..3 (b = 0..3).
template <int DP>
__device__ __forceinline__ int pa_key_swizzle(int R) { return DP == 128 ? ((R >> 1) & 1) | ((R >> 3) & 6) : (R >> 3) & 3; }
__device__ __forceinline__ int pa_value_swizzle(int R) { return (R >> 1) & 3; }

// SUB: 16-token groups of a tile on one page (pages of 16, 32 and 64 or more: 1, 2, 4)
template <typename T, int NC, int NQ, int SUB>
__global__ __launch_bounds__(256, 2) void attention_paged_kernel(const PagedArgs a)
{
    typedef Mfma<T> MM;
    typedef typename MM::vec vec;
    constexpr int MR = 16 * NQ, DP = 64 * NC, DT = 4 * NC;
    __shared__ float sm_m[4][MR], sm_l[4][MR];
    constexpr int QROW = DP + 8;   // padded row of the queries, in elements: 16 rows read side by side spread over the banks
    constexpr int NP = 4 / SUB, COPIES = DP / 16;  // pages of a tile; copy instructions (1 KB each) of its keys, of its values
    // Per wave: keys by token, values by channel.  Two objects, so that the compiler's own waits tell their copies apart.
    __shared__ __attribute__((aligned(1024))) uint8_t sm_k[4][64 * DP], sm_v[4][64 * DP];
    __shared__ __attribute__((aligned(16))) T sm_q[MR * QROW];

    const int lane = threadIdx.x & 63, m = lane & 15, g = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);   // uniform, so that what follows from it is scalar
    const int head_kv = blockIdx.x % a.n_kv_heads, split = blockIdx.y;
    const Item it = find_item(a, blockIdx.x / a.n_kv_heads, MR);
    if (it.n == 0) return;
    const int d = a.head_dim, page = 1 << a.page_log2;
    int len = it.len;
    len = len < 0 ? 0 : (len > PA_MAX_LEN ? PA_MAX_LEN : len);   // (positions and the tile behind them stay below 2^31)
    const int n_tiles = (len + 63) >> 6;
    // runs of equal length, as many as runs of tiles_per_split take (so none is longer or empty)
    const int runs = (n_tiles + a.tiles_per_split - 1) / a.tiles_per_split;
    if (split > 0 && split >= runs) return;
    const int per_run = runs > 1 && runs <= a.n_splits ? ((n_tiles + runs - 1) / runs + 3) & ~3 : a.tiles_per_split;
    const bool parts = runs > 1 && a.n_splits > 1;   // else this workgroup has the whole row
    const int t_lo = split * per_run;
    // (as far as the last of the workgroup's rows sees; a run may be empty for it)
    const int last_tok = (it.tile * MR + MR - 1) / a.group, hidden = last_tok < it.n ? it.n - 1 - last_tok : 0;
    const int vis = len > hidden ? len - hidden : 0, vis_tiles = (vis + 63) >> 6;
    const int t_hi = vis_tiles < t_lo + per_run ? vis_tiles : t_lo + per_run;

    // the query rows go to LDS (registers are what the loads in flight need), 0 where there is no row or channel
    for (int i = threadIdx.x; i < MR * DP / 8; i += 256) {
        const int rr = i / (DP / 8), ch = 8 * (i - rr * (DP / 8)), r = it.tile * MR + rr, tok = r / a.group;
        u32x4 raw = {0, 0, 0, 0};
        if (tok < it.n && ch < d)
            raw = *reinterpret_cast<const u32x4 *>((const T *)a.q + (it.row0 + tok) * a.q_tok + (int64_t)(head_kv * a.group + (r - tok * a.group)) * a.q_head + ch);
        *reinterpret_cast<u32x4 *>(&sm_q[rr * QROW + ch]) = raw;
    }
    // the last position that this lane's row (column m of each 16-row tile) sees
    int last[NQ];
#pragma unroll
    for (int nt = 0; nt < NQ; ++nt) {
        const int tok = (it.tile * MR + 16 * nt + m) / a.group;
        last[nt] = tok < it.n ? len - it.n + tok : -1;
    }
    __syncthreads();

    // The pages of a tile, in scalar registers; the entries of the table are fetched a tile before they are used.
    bool bad = vis > a.table_width << a.page_log2;   // a token that should be there lies on no page
    const int32_t *table = a.table + (int64_t)it.b * a.table_width;
    struct Pages {
        int id[NP];
    };
    const auto fetch_pages = [&](int t) {
        Pages p;
#pragma unroll
        for (int i = 0; i < NP; ++i) {
            const int tok = t * 64 + 16 * SUB * i, e = tok >> a.page_log2;
            p.id[i] = tok < vis && e < a.table_width ? pa_scalar_load(table, e) : -1;
        }
        return p;
    };
    // page 0 stands in for no page: what is read there is masked, or the row is NaN
    const auto check_pages = [&](Pages p, int t) {
#pragma unroll
        for (int i = 0; i < NP; ++i)
            if (p.id[i] < 0 || p.id[i] >= a.n_pages) {
                bad |= t * 64 + 16 * SUB * i < vis;
                p.id[i] = 0;
            }
        return p;
    };
    const int head_bytes = page * d;
    const auto copy = [&](const uint8_t *codes, int id, int off, uint8_t *to) {
        const __amdgpu_buffer_rsrc_t rs =
            __builtin_amdgcn_make_buffer_rsrc((void *)(codes + ((int64_t)id * a.n_kv_heads + head_kv) * head_bytes), 0, head_bytes, 0x00020000);
        __builtin_amdgcn_raw_ptr_buffer_load_lds(rs, GQ_LDS_PTR(void, to), 16, off, 0, 0, 0);
    };
    uint8_t *buf_k = sm_k[wave], *buf_v = sm_v[wave];
    // Copy j brings the pieces 64 j .. 64 j + 63 of the buffer, lane l piece l: of its 128 bytes R the piece that belongs
    // there.  Channels behind head_dim are out of the descriptor's range, wherever in a page the tile begins, and arrive as 0.
    constexpr int ROWS = 1024 / DP;    // tokens of a copy of keys, all on one page
    constexpr int PER = COPIES / NP;   // copies of a page's part of the tile's values: DP rows of SUB pieces
    unsigned k_off[COPIES], v_off[COPIES];   // in the page, from the tile's first token in it
#pragma unroll
    for (int j = 0; j < COPIES; ++j) {
        const int piece = (lane & 7) ^ pa_key_swizzle<DP>(8 * j + (lane >> 3));
        const int row = DP == 128 ? lane >> 3 : 2 * (lane >> 3) + (piece >> 2), ch = 16 * (DP == 128 ? piece : piece & 3);
        k_off[j] = ch < d ? ((ROWS * j) % (16 * SUB) + row) * d + ch : 0x80000000u;
        const int q = 64 * (j % PER) + (lane & ~7) + ((lane & 7) ^ pa_value_swizzle(lane >> 3)), c = q / SUB;
        v_off[j] = c < d ? c * page + 16 * (q % SUB) : 0x80000000u;
    }
    const auto copy_k = [&](int t, const Pages &p) {
        const unsigned at = SUB == 4 ? ((t * 64) & (page - 1)) * d : 0;
#pragma unroll
        for (int j = 0; j < COPIES; ++j) copy(a.k_codes, p.id[ROWS * j / (16 * SUB)], (int)(k_off[j] + at), buf_k + 1024 * j);
    };
    const auto copy_v = [&](int t, const Pages &p) {
        const unsigned at = SUB == 4 ? (t * 64) & (page - 1) : 0;
#pragma unroll
        for (int j = 0; j < COPIES; ++j) copy(a.v_codes, p.id[j / PER], (int)(v_off[j] + at), buf_v + 1024 * j);
    };
    float ks, vs, ks_next, vs_next;
    const auto load_scales = [&](const Pages &p) {
        ks_next = pa_scalar_load(a.k_scale, (int64_t)p.id[0] * a.n_kv_heads + head_kv);
        vs_next = pa_scalar_load(a.v_scale, (int64_t)p.id[0] * a.n_kv_heads + head_kv);
#pragma unroll
        for (int i = 1; i < NP; ++i) {
            const int64_t block = (int64_t)p.id[i] * a.n_kv_heads + head_kv;
            const float k1 = pa_scalar_load(a.k_scale, block), v1 = pa_scalar_load(a.v_scale, block);
            if (g >= i * SUB) {
                ks_next = k1;
                vs_next = v1;
            }
        }
    };

    f32x4 o[NQ][DT];
    float mx[NQ], l[NQ];
#pragma unroll
    for (int nt = 0; nt < NQ; ++nt) {
        mx[nt] = -INFINITY;
        l[nt] = 0.f;
#pragma unroll
        for (int t2 = 0; t2 < DT; ++t2) o[nt][t2] = f32x4{0.f, 0.f, 0.f, 0.f};
    }
    // tokens from here on are hidden from some row: behind the sequence, or after a query token of the workgroup's
    const int partly = len - it.n + it.tile * MR / a.group + 1;

    int t = t_lo + wave;
    int e0 = PA_NO_EXPONENT;   // of the first page's value scale, to which the others' are set in relation (any number is right)
    Pages next;
#pragma unroll
    for (int i = 0; i < NP; ++i) next.id[i] = 0;
    if (t < t_hi) {
        const Pages first = check_pages(fetch_pages(t), t);
        copy_k(t, first);
        copy_v(t, first);
        load_scales(first);
        if (t + 4 < t_hi) next = fetch_pages(t + 4);
    }
    const auto step = [&](auto masked, auto go_on) {
        const bool more = go_on || t + 4 < t_hi;
        ks = ks_next;
        vs = vs_next;
        Pages now = next;
        if (t + 8 < t_hi) next = fetch_pages(t + 8);
        // the keys are there: the values' copies may still be under way
        pa_wait<COPIES>();
        __builtin_amdgcn_s_setprio(1);   // a wave at its products goes before one at its exponentials (1 x 131071: 74.2 -> 73.4 us)
        f32x4 s[NQ][4];
#pragma unroll
        for (int nt = 0; nt < NQ; ++nt)
#pragma unroll
            for (int i = 0; i < 4; ++i) s[nt][i] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int c = 0; c < NC; ++c) {
            u32x4 kr[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int row = 16 * (m >> 2) + 4 * i + (m & 3), R = DP == 128 ? row : row >> 1, piece = DP == 128 ? 4 * c + g : 4 * (row & 1) + g;
                kr[i] = *reinterpret_cast<const u32x4 *>(buf_k + 128 * R + 16 * (piece ^ pa_key_swizzle<DP>(R)));
            }
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                vec qf[NQ];
#pragma unroll
                for (int nt = 0; nt < NQ; ++nt) qf[nt] = *reinterpret_cast<const vec *>(&sm_q[(16 * nt + m) * QROW + 64 * c + 16 * g + 8 * h]);
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const vec kf = MM::decode(kr[i][2 * h], kr[i][2 * h + 1]);
#pragma unroll
                    for (int nt = 0; nt < NQ; ++nt) s[nt][i] = MM::run(kf, qf[nt], s[nt][i]);
                }
            }
        }
        __builtin_amdgcn_s_setprio(0);
        if (more) {
            now = check_pages(now, t + 4);
            pa_reads_done();
            copy_k(t + 4, now);
            load_scales(now);
        }
        vs = vs < 0x1p-100f ? 0x1p-100f : vs;   // a scale of 0 must not become an infinite weight, one that is NaN stays it
        int e = pa_exponent(vs);
        if (e0 == PA_NO_EXPONENT) {   // (here, where the scale has long arrived: before the loop it cost single tokens 0.3 us)
            e0 = __builtin_amdgcn_readfirstlane(e);
            e0 = e0 < -80 ? -80 : (e0 > 100 ? 100 : e0);   // the scale of a page of zeros is 2^-100: 2^e / vs stays far from 2^128
        }
        e -= e0;
        e = e < -15 ? -15 : (e > 7 ? 7 : e);
        const float unit = __uint_as_float((unsigned)(e + 127) << 23);
        const float mul = a.scale * ks, add = __builtin_amdgcn_logf(vs) - (float)e, inv = unit / vs;
        f16x8 p[NQ][2];
#pragma unroll
        for (int nt = 0; nt < NQ; ++nt) {
            float top = -INFINITY;
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    if constexpr (masked) {
                        const float y = fmaf(s[nt][i][j], mul, add);
                        s[nt][i][j] = t * 64 + 16 * g + 4 * i + j > last[nt] ? -INFINITY : y;
                    }
                    top = fmaxf(top, s[nt][i][j]);
                }
            if constexpr (!masked) top = fmaf(top, mul, add);   // (a lane's tokens have one scale, and it is positive)
            top = gq_max_xor32(gq_max_xor16(top));
            // M follows the maximum only when that is more than 8 above it: O is rescaled in a wave's first tile instead of in
            // most (some row of 16 finds a new maximum in nearly every one; 1 x 131071: 74.5 -> 74.1 us)
            if (__any(top > mx[nt] + 8.f)) {
                const float to = fmaxf(top, mx[nt]);
                const float f = mx[nt] == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(mx[nt] - to);
                mx[nt] = to;
                l[nt] *= f;
#pragma unroll
                for (int t2 = 0; t2 < DT; ++t2)
#pragma unroll
                    for (int j = 0; j < 4; ++j) o[nt][t2][j] *= f;
            }
            const float ref = mx[nt] == -INFINITY ? 0.f : mx[nt] - 7.f;
            float sum = 0.f;
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const float w = __builtin_amdgcn_exp2f(masked ? s[nt][i][j] - ref : fmaf(s[nt][i][j], mul, add - ref));
                    sum += w;
                    p[nt][i >> 1][4 * (i & 1) + j] = (_Float16)w;
                }
            // (where a lane sees none of its tokens, their page's scale may be anything, NaN too)
            l[nt] = masked && sum == 0.f ? l[nt] : fmaf(sum, inv, l[nt]);
        }
        if (more) pa_wait<COPIES>();   // the values are there: the next keys may be under way
        else pa_wait<0>();
        u32x4 vr[DT];
#pragma unroll
        for (int t2 = 0; t2 < DT; ++t2) {
            const int q = (16 * t2 + m) * SUB + g % SUB, R = q >> 3;
            vr[t2] = *reinterpret_cast<const u32x4 *>(buf_v + (g / SUB) * (DP * SUB * 16) + 128 * R + 16 * ((q & 7) ^ pa_value_swizzle(R)));
        }
        bool apart = false;   // a NaN among the values of a tile that is not visible to every row
        if (masked) {
            const int left = len - (t * 64 + 16 * g);   // of this lane's 16 tokens
            bool nan = false;
#pragma unroll
            for (int t2 = 0; t2 < DT; ++t2)
#pragma unroll
                for (int w = 0; w < 4; ++w) {
                    const int k = left - 4 * w;
                    const unsigned keep = k >= 4 ? 0xffffffffu : (k <= 0 ? 0u : (1u << (8 * k)) - 1);
                    const unsigned x = vr[t2][w] & keep;
                    vr[t2][w] = x;
                    // a byte is NaN where its low seven bits are all set: then adding 1 carries into the eighth
                    nan |= (((x & 0x7f7f7f7fu) + 0x01010101u) & 0x80808080u) != 0;
                }
            apart = it.n > 1 && __any(nan);
        }
        if (!apart) {
            __builtin_amdgcn_s_setprio(1);
#pragma unroll
            for (int t2 = 0; t2 < DT; ++t2) {
#pragma unroll
                for (int u = 0; u < 2; ++u) {
                    const f16x8 vf = Mfma<_Float16>::decode(vr[t2][2 * u], vr[t2][2 * u + 1], unit);
#pragma unroll
                    for (int nt = 0; nt < NQ; ++nt) o[nt][t2] = Mfma<_Float16>::run(vf, p[nt][u], o[nt][t2]);
                }
            }
        } else {
            // 0 * NaN is NaN: one token at a time, added only to the rows that see it
            for (int tok = 0; tok < 64; ++tok) {
                if (t * 64 + tok >= len) break;
#pragma unroll
                for (int t2 = 0; t2 < DT; ++t2) {
                    unsigned w[4];
#pragma unroll
                    for (int i = 0; i < 4; ++i)
                        w[i] = (tok >> 4) == g && ((tok >> 2) & 3) == i ? vr[t2][i] & (0xffu << (8 * (tok & 3))) : 0u;
#pragma unroll
                    for (int nt = 0; nt < NQ; ++nt) {
                        f32x4 x = Mfma<_Float16>::run(Mfma<_Float16>::decode(w[0], w[1], unit), p[nt][0], f32x4{0.f, 0.f, 0.f, 0.f});
                        x = Mfma<_Float16>::run(Mfma<_Float16>::decode(w[2], w[3], unit), p[nt][1], x);
                        if (t * 64 + tok <= last[nt]) o[nt][t2] += x;
                    }
                }
            }
        }
        __builtin_amdgcn_s_setprio(0);
        if (more) {
            pa_reads_done();
            copy_v(t + 4, now);
        }
        t += 4;
    };
    // (the first loop without a branch around the copies: a wait the compiler adds has to know what is under way)
    while ((t + 1) * 64 <= partly && t + 4 < t_hi) step(std::false_type(), std::true_type());
    while (t < t_hi) step(std::true_type(), std::false_type());

    // join the four waves, through the keys' buffers: a row's 16-byte pieces are permuted by the row, for the banks
    float *sm_o = reinterpret_cast<float *>(&sm_k[0][0]);
    const auto o_at = [&](int w, int row, int ch) { return reinterpret_cast<f32x4 *>(sm_o + (w * 16 + row) * DP + 4 * ((ch >> 2) ^ row)); };
    const bool any_bad = __any(bad);
#pragma unroll
    for (int nt = 0; nt < NQ; ++nt) {
        l[nt] += __shfl_xor(l[nt], 16, 64);
        l[nt] += __shfl_xor(l[nt], 32, 64);
        if (any_bad) l[nt] = NAN;
        if (g == 0) {
            sm_m[wave][16 * nt + m] = mx[nt];
            sm_l[wave][16 * nt + m] = l[nt];
        }
    }
    __syncthreads();
#pragma unroll
    for (int nt = 0; nt < NQ; ++nt) {
        const int rm = 16 * nt + m;
        const float all = fmaxf(fmaxf(sm_m[0][rm], sm_m[1][rm]), fmaxf(sm_m[2][rm], sm_m[3][rm]));
        const float f = mx[nt] == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(mx[nt] - all);
        if (nt > 0) __syncthreads();   // (before the first, all waves are done with their tiles)
#pragma unroll
        for (int t2 = 0; t2 < DT; ++t2) {
            f32x4 x = o[nt][t2];
#pragma unroll
            for (int j = 0; j < 4; ++j) x[j] *= f;
            *o_at(wave, m, 16 * t2 + 4 * g) = x;
        }
        __syncthreads();
        const int row = threadIdx.x >> 4, rr = 16 * nt + row, r = it.tile * MR + rr, tok = r / a.group;
        if (tok >= it.n) continue;
        const float ma = fmaxf(fmaxf(sm_m[0][rr], sm_m[1][rr]), fmaxf(sm_m[2][rr], sm_m[3][rr]));
        float sum = 0.f;
        for (int w = 0; w < 4; ++w) sum += sm_l[w][rr] * (sm_m[w][rr] == -INFINITY ? (sm_l[w][rr] == 0.f ? 0.f : 1.f) : __builtin_amdgcn_exp2f(sm_m[w][rr] - ma));
        const int head = head_kv * a.group + (r - tok * a.group);
        const int64_t qrow = it.row0 + tok;
        for (int ch = 4 * (threadIdx.x & 15); ch < d; ch += 64) {
            f32x4 x = {0.f, 0.f, 0.f, 0.f};
            for (int w = 0; w < 4; ++w) x += *o_at(w, row, ch);
            if (parts) {
                *reinterpret_cast<f32x4 *>(a.part_o + ((qrow * a.n_heads + head) * a.n_splits + split) * d + ch) = x;
            } else {
                // a row without a key is 0
                T y[4];
                for (int j = 0; j < 4; ++j) y[j] = (T)(sum == 0.f ? 0.f : x[j] / sum);
                u32x2 raw;
                __builtin_memcpy(&raw, y, 8);
                *reinterpret_cast<u32x2 *>((T *)a.out + qrow * a.o_tok + (int64_t)head * a.o_head + ch) = raw;
            }
        }
        if (parts && (threadIdx.x & 15) == 0) {
            float *ml = a.part_ml + ((qrow * a.n_heads + head) * a.n_splits + split) * 2;
            ml[0] = ma;
            ml[1] = sum;
        }
    }
}

// Joins a row's partial results: O = sum_s 2^(M_s - M) O_s / sum_s 2^(M_s - M) l_s.  One workgroup per row: 8 groups of
// 32 lanes take every eighth run (4 channels a lane), so that a row of many runs is few loads deep.
template <typename T>
__global__ __launch_bounds__(256) void attention_paged_join_kernel(const PagedArgs a)
{
    __shared__ float sm_f[PA_MAX_SPLITS], sm_sum;
    __shared__ f32x4 sm_x[8][32];
    const int64_t idx = blockIdx.x, tok = idx / a.n_heads;
    const int head = (int)(idx - tok * a.n_heads), tid = threadIdx.x, part = tid >> 5, ch = 4 * (tid & 31);
    int b = (int)tok;
    if (a.cu) {
        if (tok < a.cu[0] || tok >= a.cu[a.batch]) return;   // behind the last sequence: left as it is
        int lo = -1;
        for (int b0 = 0; b0 < a.batch; b0 += 64) {
            const int c = __popcll(__ballot(b0 + (tid & 63) < a.batch && a.cu[b0 + (tid & 63)] <= tok));
            lo += c;
            if (c < 64) break;
        }
        lo = __builtin_amdgcn_readfirstlane(lo < 0 ? 0 : lo);
        b = lo;
        if (a.cu[b + 1] <= tok || a.cu[b] < 0 || a.cu[b + 1] > a.n_tokens) return;   // not rising: the first kernel left it out
    }
    const int len = a.lens[b] < 0 ? 0 : (a.lens[b] > PA_MAX_LEN ? PA_MAX_LEN : a.lens[b]);
    const int wanted = ((len + 63) / 64 + a.tiles_per_split - 1) / a.tiles_per_split;
    if (wanted <= 1) return;   // one run: the first kernel wrote the row
    const int used = wanted > a.n_splits ? a.n_splits : wanted;
    if (tid < 64) {   // PA_MAX_SPLITS runs at most: one wave weighs them
        const float *ml = a.part_ml + (idx * a.n_splits + tid) * 2;
        const float mx = tid < used ? ml[0] : -INFINITY, l = tid < used ? ml[1] : 0.f;
        float top = mx;
#pragma unroll
        for (int off = 32; off > 0; off >>= 1) top = fmaxf(top, __shfl_xor(top, off, 64));
        const float f = mx == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(mx - top);
        float sum = mx == -INFINITY ? l : l * f;   // (0 without a key, NaN for a bad table)
#pragma unroll
        for (int off = 32; off > 0; off >>= 1) sum += __shfl_xor(sum, off, 64);
        sm_f[tid] = f;
        // more tokens than the table has pages for
        if (tid == 0) sm_sum = wanted > a.n_splits ? NAN : sum;
    }
    __syncthreads();
    f32x4 x = {0.f, 0.f, 0.f, 0.f};
    if (ch < a.head_dim)
        for (int s = part; s < used; s += 8) {
            const f32x4 v = *reinterpret_cast<const f32x4 *>(a.part_o + (idx * a.n_splits + s) * a.head_dim + ch);
            const float f = sm_f[s];
#pragma unroll
            for (int j = 0; j < 4; ++j) x[j] = fmaf(v[j], f, x[j]);
        }
    sm_x[part][tid & 31] = x;
    __syncthreads();
    if (part == 0 && ch < a.head_dim) {
#pragma unroll
        for (int p = 1; p < 8; ++p) x += sm_x[p][tid];
        const float sum = sm_sum;
        T y[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) y[j] = (T)(sum == 0.f ? 0.f : x[j] / sum);
        u32x2 raw;
        __builtin_memcpy(&raw, y, 8);
        *reinterpret_cast<u32x2 *>((T *)a.out + tok * a.o_tok + (int64_t)head * a.o_head + ch) = raw;
    }
}

struct Plan {
    int nq, n_splits, tiles_per_split;
    int64_t n_items;
};

// Query rows per workgroup: one or two 16-row tiles (four do not fit the registers of two waves a SIMD).  Two where there are
// more rows than one holds: 512 tokens behind 7680 with one and with two tiles 274 and 199 us, four tokens of one sequence of
// 131071 75.2 and 73.7; on batches that one tile reads often enough two cost a little (8 sequences of 2048 with eight tokens
// each 30.2 and 33).  One for 16 rows or fewer: 16 tokens of 8 sequences of 2048, 32 heads of their own, 35.4 and 42.3, single
// tokens 131 and 145.
// Runs: workgroups for two rounds (512 run at once), of at least 256 tokens (one tile per wave), at most 64 of them.  Sequences of
// 4096, 2048 and 8192 tokens 108, 98 and 107 us; with twice as many 113, 115 and 110, with half as many 97, 98 and 105; 64 of
// 391 to 8192 tokens 132, 132 and 129 (operands that no cache holds).
Plan paged_plan(int64_t n_tokens, int64_t batch, bool ragged, int64_t n_heads, int64_t n_kv_heads, int64_t page, int64_t table_width)
{
    Plan p;
    const int64_t group = n_heads / n_kv_heads;
    const int64_t rows = ragged ? gq_cdiv(n_tokens * group, batch) : group;
    p.nq = rows <= 16 ? 1 : 2;
    const int mr = 16 * p.nq;
    p.n_items = ragged ? n_tokens * group / mr + batch : batch * gq_cdiv(group, mr);
    const int64_t tiles = gq_cdiv(table_width * page, 64), wgs = p.n_items * n_kv_heads;
    int64_t splits = gq_cdiv(1024, wgs);
    splits = std::min<int64_t>(splits, gq_cdiv(tiles, 4));
    splits = std::max<int64_t>(1, std::min<int64_t>(splits, PA_MAX_SPLITS));
    p.tiles_per_split = (int)std::max<int64_t>(4, gq_round_up(gq_cdiv(tiles, splits), 4));
    p.n_splits = (int)std::max<int64_t>(1, gq_cdiv(tiles, p.tiles_per_split));
    return p;
}

bool paged_sizes_ok(int64_t n_tokens, int64_t batch, int64_t n_heads, int64_t n_kv_heads, int64_t head_dim, int64_t page, int64_t table_width)
{
    return n_tokens >= 0 && n_tokens < ((int64_t)1 << 31) && batch >= 0 && batch < (1 << 24) && n_kv_heads > 0 && n_heads > 0 && n_heads <= 65536 &&
           n_heads % n_kv_heads == 0 && head_dim >= 16 && head_dim <= 128 && head_dim % 16 == 0 &&
           (page == 16 || page == 32 || page == 64 || page == 128) && table_width >= 0 && table_width * page < PA_MAX_LEN;
}

template <typename T>
int launch_paged(const PagedArgs &a, const Plan &p, hipStream_t s)
{
    const dim3 grid((unsigned)(p.n_items * a.n_kv_heads), (unsigned)p.n_splits);
#define GQ_PA(NC, NQ)                                                                                                       \
    do {                                                                                                                    \
        if (a.page_log2 >= 6) hipLaunchKernelGGL((attention_paged_kernel<T, NC, NQ, 4>), grid, dim3(256), 0, s, a);         \
        else if (a.page_log2 == 5) hipLaunchKernelGGL((attention_paged_kernel<T, NC, NQ, 2>), grid, dim3(256), 0, s, a);    \
        else hipLaunchKernelGGL((attention_paged_kernel<T, NC, NQ, 1>), grid, dim3(256), 0, s, a);                          \
    } while (0)
    if (a.head_dim <= 64) {
        if (p.nq == 1) GQ_PA(1, 1);
        else GQ_PA(1, 2);
    } else {
        if (p.nq == 1) GQ_PA(2, 1);
        else GQ_PA(2, 2);
    }
#undef GQ_PA
    GQ_LAUNCH_CHECK();
    if (p.n_splits > 1) {
        hipLaunchKernelGGL(attention_paged_join_kernel<T>, dim3((unsigned)(a.n_tokens * a.n_heads)), dim3(256), 0, s, a);
        GQ_LAUNCH_CHECK();
    }
    return GQ_OK;
}

}  // namespace

extern "C" size_t gq_attention_paged_workspace(int64_t n_tokens, int64_t batch, int ragged, int n_heads, int n_kv_heads, int head_dim, int page,
                                               int64_t table_width)
{
    if (!paged_sizes_ok(n_tokens, batch, n_heads, n_kv_heads, head_dim, page, table_width) || n_tokens == 0 || batch == 0) return 0;
    const Plan p = paged_plan(n_tokens, batch, ragged != 0, n_heads, n_kv_heads, page, table_width);
    return p.n_splits == 1 ? 0 : (size_t)n_tokens * n_heads * p.n_splits * (head_dim + 4) * sizeof(float);
}

extern "C" int gq_attention_paged(const gq_attention_paged_args *args, gq_stream_t stream)
{
    GQ_REQUIRE(args, "gq_attention_paged: NULL pointer");
    const gq_paged_cache cache = args->cache;
    const gq_rows out = args->out, q = args->q;
    const int64_t dtype = args->dtype, n_tokens = args->n_tokens, n_heads = args->n_heads, n_pages = cache.n_pages, n_kv_heads = cache.n_kv_heads;
    const int64_t page = cache.page, head_dim = cache.head_dim, table_width = args->table_width, batch = args->batch;
    const int32_t *block_table = args->block_table, *seq_lens = args->seq_lens, *cu_seqlens = args->cu_seqlens;
    const float softmax_scale = (float)args->softmax_scale;
    void *workspace = args->workspace;
    const size_t workspace_bytes = args->workspace_bytes < 0 ? 0 : (size_t)args->workspace_bytes;
    GQ_REQUIRE(dtype == GQ_F16 || dtype == GQ_BF16, "gq_attention_paged: dtype %lld is neither fp16 (0) nor bf16 (1)", (long long)dtype);
    GQ_REQUIRE(paged_sizes_ok(n_tokens, batch, n_heads, n_kv_heads, head_dim, page, table_width) && n_pages >= 0,
               "gq_attention_paged: %lld heads on %lld, head_dim %lld (a multiple of 16 up to 128), pages of %lld (16, 32, 64 or 128): not supported",
               (long long)n_heads, (long long)n_kv_heads, (long long)head_dim, (long long)page);
    GQ_REQUIRE(cu_seqlens || n_tokens == batch, "gq_attention_paged: %lld tokens for %lld sequences need cu_seqlens", (long long)n_tokens,
               (long long)batch);
    GQ_REQUIRE(softmax_scale > 0.f && softmax_scale * PA_LOG2E < INFINITY, "gq_attention_paged: the softmax scale must be positive and finite");
    if (n_tokens == 0 || batch == 0) return GQ_OK;
    GQ_REQUIRE(out.data && q.data && seq_lens && (table_width == 0 || block_table) && cache.k_codes && cache.v_codes && cache.k_scale && cache.v_scale,
               "gq_attention_paged: NULL pointer");
    GQ_REQUIRE(q.token_stride % 8 == 0 && q.head_stride % 8 == 0 && out.token_stride % 8 == 0 && out.head_stride % 8 == 0,
               "gq_attention_paged: strides must be multiples of 8 elements");
    GQ_REQUIRE(gq_rows_apart(out, n_tokens, n_heads, head_dim), "gq_attention_paged: rows of out overlap");
    GQ_REQUIRE((((uintptr_t)out.data | (uintptr_t)q.data | (uintptr_t)cache.k_codes | (uintptr_t)cache.v_codes | (uintptr_t)workspace) & 15) == 0,
               "gq_attention_paged: pointers must be 16-byte aligned");
    const Plan p = paged_plan(n_tokens, batch, cu_seqlens != nullptr, n_heads, n_kv_heads, page, table_width);
    GQ_REQUIRE(n_pages > 0, "gq_attention_paged: a cache without pages");
    GQ_REQUIRE(n_pages < ((int64_t)1 << 31) && p.n_items * n_kv_heads < GQ_MAX_THREADS / 256 && n_tokens * n_heads < ((int64_t)1 << 31), "gq_attention_paged: too many query rows for one call");
    const size_t need = p.n_splits == 1 ? 0 : (size_t)n_tokens * n_heads * p.n_splits * (head_dim + 4) * sizeof(float);
    if (workspace_bytes < need || (need && !workspace)) {
        gq_set_error("gq_attention_paged: workspace of %zu bytes, %zu needed", workspace_bytes, need);
        return GQ_EWORKSPACE;
    }
    PagedArgs a;
    a.q = q.data, a.out = out.data, a.q_tok = q.token_stride, a.q_head = q.head_stride, a.o_tok = out.token_stride, a.o_head = out.head_stride;
    a.k_codes = (const uint8_t *)cache.k_codes, a.v_codes = (const uint8_t *)cache.v_codes, a.k_scale = cache.k_scale, a.v_scale = cache.v_scale;
    a.table = block_table, a.lens = seq_lens, a.cu = cu_seqlens;
    a.part_o = (float *)workspace;
    a.part_ml = (float *)workspace + (size_t)n_tokens * n_heads * p.n_splits * head_dim;
    a.n_tokens = n_tokens, a.n_pages = (int)n_pages, a.table_width = (int)table_width;
    a.batch = (int)batch, a.n_heads = (int)n_heads, a.n_kv_heads = (int)n_kv_heads, a.group = (int)(n_heads / n_kv_heads), a.head_dim = (int)head_dim;
    a.page_log2 = __builtin_ctz((unsigned)page), a.tiles_per_split = p.tiles_per_split, a.n_splits = p.n_splits, a.n_items = (int)p.n_items;
    a.scale = softmax_scale * PA_LOG2E;
    return dtype == GQ_F16 ? launch_paged<_Float16>(a, p, (hipStream_t)stream) : launch_paged<__bf16>(a, p, (hipStream_t)stream);
}
