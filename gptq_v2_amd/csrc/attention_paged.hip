// Attention of a few query tokens per sequence over a paged cache of 8-bit keys and values (the layout and the scales
// that kv_append.hip writes): a decoder's step for one new token, or for the several of a checked draft or a chunk.
//
// With K = ks[page] k8 and V = vs[page] v8, in powers of two (c = softmax scale * log2 e):
//   y_t = c ks (q . k8_t) + log2 vs,  M = max y,  w_t = 2^(y_t - M),  O = sum_t w_t v8_t / sum_t w_t / vs
// The value's scale sits in the exponent, so the weights that meet the codes on the matrix core are at most 1 whatever
// the scales are, and the denominator takes it out again in 32 bits.
//
// A wave takes 64 tokens at a time, all from registers: S^T = K Q^T (16 x 16 x 32 tiles: tokens by query rows) and
// O^T = V^T P^T.  Row 4 g + i of the S^T tile a stands for token 16 g + 4 a + i; lane group g then holds, as the tiles'
// results, the weights of the 16 adjacent tokens 16 g .. 16 g + 15 of its query row -- exactly what it has to supply as
// the operand P^T, and exactly the 16 bytes it loads of a row of V^T.  No value crosses lanes but for the maximum.
// The rows are the query heads that share a kv head (times the tokens of the sequence); the cache is read once for
// every 16 NQ of them.  e4m3 codes are exact in either 16-bit type: Q K^T runs in q's type, P V in fp16 (w <= 1 keeps
// 11 bits there, against 8 in bf16).
//
// Bound by HBM: 2 head_dim bytes per cached token and kv head.  A long sequence is cut into runs of tokens for several
// workgroups, whose (O, M, l) a second kernel joins.
#include <type_traits>

#include "gq_common.h"

namespace {

constexpr int PA_MAX_SPLITS = 64;   // one wave weighs them
constexpr int PA_MAX_LEN = 1 << 30;     // longest sequence; tables are narrower (a longer one is NaN)
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

typedef __amdgpu_buffer_rsrc_t pa_rsrc_t;

template <typename T> struct Mfma;
template <> struct Mfma<_Float16> {
    typedef f16x8 vec;
    static __device__ __forceinline__ f32x4 run(f16x8 a, f16x8 b, f32x4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0); }
    // 8 codes (two words) to the operand's type, exactly
    static __device__ __forceinline__ f16x8 decode(unsigned lo, unsigned hi)
    {
        const f16x2 a = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(lo, 1.f, false), b = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(lo, 1.f, true);
        const f16x2 c = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(hi, 1.f, false), d = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(hi, 1.f, true);
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
};

__device__ __forceinline__ Item find_item(const PagedArgs &a, int item, int mr)
{
    if (!a.cu) {
        const int tiles = (a.group + mr - 1) / mr;
        const int b = item / tiles;
        return {b, item - b * tiles, b, 1};
    }
    const auto start = [&](int s) { return (int64_t)a.cu[s] * a.group / mr + s; };
    int lo = 0, hi = a.batch - 1;
    while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (start(mid) <= item) lo = mid;
        else hi = mid - 1;
    }
    const int64_t row0 = a.cu[lo], n = (int64_t)a.cu[lo + 1] - row0, tile = item - start(lo);
    if (row0 < 0 || n <= 0 || row0 + n > a.n_tokens || tile < 0 || tile * mr >= n * a.group) return {lo, 0, 0, 0};
    return {lo, (int)tile, row0, (int)n};
}

// ONE: a tile of 64 tokens lies on one page (pages of 64 or 128), whose address is then the same for all lanes: a scalar
// descriptor and 32-bit lane offsets instead of 64-bit addresses per lane and load.
template <typename T, int NC, int NQ, bool ONE>
__global__ __launch_bounds__(256, NQ == 1 ? 3 : (NQ == 2 ? 2 : 1)) void attention_paged_kernel(const PagedArgs a)
{
    typedef Mfma<T> MM;
    typedef typename MM::vec vec;
    constexpr int MR = 16 * NQ, DP = 64 * NC, DT = 4 * NC;
    constexpr int LROW = DP + 4;   // padded row of the join buffer, in floats
    __shared__ float sm_m[4][MR], sm_l[4][MR];
    constexpr int QROW = DP + 8;   // padded row of the queries, in elements: 16 rows read side by side spread over the banks
    union Shared {
        float o[4][16 * LROW];
        T q[MR * QROW];
    };
    __shared__ __attribute__((aligned(16))) Shared sm;

    const int lane = threadIdx.x & 63, m = lane & 15, g = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);   // uniform, so that what follows from it is scalar
    const int head_kv = blockIdx.x % a.n_kv_heads, split = blockIdx.y;
    const Item it = find_item(a, blockIdx.x / a.n_kv_heads, MR);
    if (it.n == 0) return;
    const int d = a.head_dim, page = 1 << a.page_log2;
    int len = a.lens[it.b];
    len = len < 0 ? 0 : (len > PA_MAX_LEN ? PA_MAX_LEN : len);   // (positions and the tile behind them stay below 2^31)
    const int n_tiles = (len + 63) >> 6;
    const int t_lo = split * a.tiles_per_split;
    const int t_hi = n_tiles < t_lo + a.tiles_per_split ? n_tiles : t_lo + a.tiles_per_split;
    if (split > 0 && t_lo >= n_tiles) return;

    // the query rows go to LDS (registers are what the loads in flight need), 0 where there is no row or channel
    for (int i = threadIdx.x; i < MR * DP / 8; i += 256) {
        const int rr = i / (DP / 8), ch = 8 * (i - rr * (DP / 8)), r = it.tile * MR + rr, tok = r / a.group;
        u32x4 raw = {0, 0, 0, 0};
        if (tok < it.n && ch < d)
            raw = *reinterpret_cast<const u32x4 *>((const T *)a.q + (it.row0 + tok) * a.q_tok + (int64_t)(head_kv * a.group + (r - tok * a.group)) * a.q_head + ch);
        *reinterpret_cast<u32x4 *>(&sm.q[rr * QROW + ch]) = raw;
    }
    // the last position that this lane's row (column m of each 16-row tile) sees
    int last[NQ];
#pragma unroll
    for (int nt = 0; nt < NQ; ++nt) {
        const int tok = (it.tile * MR + 16 * nt + m) / a.group;
        last[nt] = tok < it.n ? len - it.n + tok : -1;
    }
    __syncthreads();

    // The pages of a tile of 64 tokens from this lane's two points of view: of the keys of tokens 16 (m / 4).. and of
    // the values of tokens 16 g.. (ONE: the same for all, in scalar registers).  The entries of the table are fetched a
    // tile before they are used, and in front of that tile's loads: waits are for loads in the order they were issued.
    bool bad = false;   // a token that should be there lies on no page
    const int32_t *table = a.table + (int64_t)it.b * a.table_width;
    struct Pages {
        int k, v;
    };
    const auto entry = [&](int tok) {
        const int i = tok >> a.page_log2;
        return tok < len && i < a.table_width ? table[i] : -1;
    };
    const auto fetch_pages = [&](int t) -> Pages {
        if constexpr (ONE) {
            const int id = entry(t * 64);
            return {id, id};
        } else {
            return {entry(t * 64 + 16 * (m >> 2)), entry(t * 64 + 16 * g)};
        }
    };
    // page 0 stands in for no page
    const auto check_pages = [&](Pages p, int t) -> Pages {
        const auto one = [&](int id, int tok) {
            if (id >= 0 && id < a.n_pages) return id;
            bad |= tok < len;
            return 0;
        };
        if constexpr (ONE) {
            const int id = one(p.k, t * 64);
            return {id, id};
        } else {
            return {one(p.k, t * 64 + 16 * (m >> 2)), one(p.v, t * 64 + 16 * g)};
        }
    };
    // What lies behind the sequence, on no page or behind head_dim is read from a place that exists (page 0, the row's
    // first channels, the first channels' rows) and does not count: such scores are masked or met by zeros of q, such
    // values are cleared or their results not written.
    const int head_bytes = page * d;
    // The lane's offsets are worked out anew for each tile (from a lane number the compiler does not see through): kept
    // over the loop they are the first thing it spills, and a reload waits for every load in flight.
    const auto lane_again = [&]() {
        int x = lane;
        asm volatile("" : "+v"(x));
        return x;
    };
    const auto k_offset = [&](int l, int c) {
        const int mm = l & 15, gg = l >> 4;
        return (unsigned)((mm & 3) * d + (ONE ? 16 * (mm >> 2) * d : 0) + (64 * c + 16 * gg < d ? 64 * c + 16 * gg : 0));
    };
    u32x4 kr[4][NC], vr[DT];
    float ks, vs, ks_next, vs_next;
    // ONE: a buffer descriptor of the page's block (scalar), 32-bit lane offsets
    const auto block_of = [&](const uint8_t *codes, int id) {
        return __builtin_amdgcn_make_buffer_rsrc((void *)(codes + ((int64_t)id * a.n_kv_heads + head_kv) * head_bytes), 0, head_bytes, 0x00020000);
    };
    const auto load_k = [&](int t, int id) {
        const int l = lane_again();
        unsigned k_off[NC];
#pragma unroll
        for (int c = 0; c < NC; ++c) k_off[c] = k_offset(l, c);
        if constexpr (ONE) {
            const pa_rsrc_t rs = block_of(a.k_codes, id);
            const int at = ((t * 64) & (page - 1)) * d;
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
                for (int c = 0; c < NC; ++c) kr[i][c] = __builtin_amdgcn_raw_buffer_load_b128(rs, (int)k_off[c], at + 4 * i * d, 0);
        } else {
            const uint8_t *p = a.k_codes + ((int64_t)id * a.n_kv_heads + head_kv) * head_bytes + ((t * 64 + 16 * (m >> 2)) & (page - 1)) * d;
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
                for (int c = 0; c < NC; ++c) kr[i][c] = *reinterpret_cast<const u32x4 *>(p + 4 * i * d + k_off[c]);
        }
    };
    const auto load_v = [&](int t, int id) {
        const int l = lane_again();
        const unsigned v_off = (l & 15) * page + (ONE ? 16 * (l >> 4) : 0);
        if constexpr (ONE) {
            const pa_rsrc_t rs = block_of(a.v_codes, id);
            const int at = (t * 64) & (page - 1);
#pragma unroll
            for (int t2 = 0; t2 < DT; ++t2) vr[t2] = __builtin_amdgcn_raw_buffer_load_b128(rs, (int)v_off, at + (16 * t2 < d ? 16 * t2 * page : 0), 0);
        } else {
            const uint8_t *p = a.v_codes + ((int64_t)id * a.n_kv_heads + head_kv) * head_bytes + ((t * 64 + 16 * g) & (page - 1));
#pragma unroll
            for (int t2 = 0; t2 < DT; ++t2) vr[t2] = *reinterpret_cast<const u32x4 *>(p + (16 * t2 < d ? 16 * t2 * page : 0) + v_off);
        }
    };
    const auto load_scales = [&](int id) {
        const int64_t block = (int64_t)id * a.n_kv_heads + head_kv;
        ks_next = a.k_scale[block];
        vs_next = a.v_scale[block];
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
    // tokens from here on are hidden from some row: behind the sequence, or after a query token of it
    const int partly = len - it.n + 1;

    // One set of registers: the next tile's keys are loaded as soon as this one's have met the queries, its values after
    // this one's have met the weights.
    int t = t_lo + wave;
    Pages next = {0, 0};
    if (t < t_hi) {
        const Pages first = check_pages(fetch_pages(t), t);
        if (t + 4 < t_hi) next = fetch_pages(t + 4);
        load_k(t, first.k);
        load_v(t, first.v);
        load_scales(first.v);
    }
    const auto step = [&](auto masked) {
        const bool more = t + 4 < t_hi;
        ks = ks_next;
        vs = vs_next;
        Pages now = next;
        if (t + 8 < t_hi) next = fetch_pages(t + 8);
        f32x4 s[NQ][4];
#pragma unroll
        for (int nt = 0; nt < NQ; ++nt)
#pragma unroll
            for (int i = 0; i < 4; ++i) s[nt][i] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int c = 0; c < NC; ++c)
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                vec qf[NQ];
#pragma unroll
                for (int nt = 0; nt < NQ; ++nt) qf[nt] = *reinterpret_cast<const vec *>(&sm.q[(16 * nt + m) * QROW + 64 * c + 16 * g + 8 * h]);
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const vec kf = MM::decode(kr[i][c][2 * h], kr[i][c][2 * h + 1]);
#pragma unroll
                    for (int nt = 0; nt < NQ; ++nt) s[nt][i] = MM::run(kf, qf[nt], s[nt][i]);
                }
                __builtin_amdgcn_sched_barrier(0);
            }
        if (more) {
            now = check_pages(now, t + 4);
            load_k(t + 4, now.k);
            load_scales(now.v);
        }
        vs = fmaxf(vs, 1e-30f);   // a scale of 0 must not become an infinite weight
        const float mul = a.scale * ks, add = __builtin_amdgcn_logf(vs), inv = 1.f / vs;
        f16x8 p[NQ][2];
#pragma unroll
        for (int nt = 0; nt < NQ; ++nt) {
            float top = -INFINITY;
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    float y = fmaf(s[nt][i][j], mul, add);
                    if (masked && t * 64 + 16 * g + 4 * i + j > last[nt]) y = -INFINITY;
                    s[nt][i][j] = y;
                    top = fmaxf(top, y);
                }
            top = fmaxf(top, __shfl_xor(top, 16, 64));
            top = fmaxf(top, __shfl_xor(top, 32, 64));
            if (__any(top > mx[nt])) {
                const float to = fmaxf(top, mx[nt]);
                const float f = mx[nt] == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(mx[nt] - to);
                mx[nt] = to;
                l[nt] *= f;
#pragma unroll
                for (int t2 = 0; t2 < DT; ++t2)
#pragma unroll
                    for (int j = 0; j < 4; ++j) o[nt][t2][j] *= f;
            }
            const float ref = mx[nt] == -INFINITY ? 0.f : mx[nt];
            float sum = 0.f;
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const float w = __builtin_amdgcn_exp2f(s[nt][i][j] - ref);
                    sum += w;
                    p[nt][i >> 1][4 * (i & 1) + j] = (_Float16)w;
                }
            l[nt] = fmaf(sum, inv, l[nt]);
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
#pragma unroll
            for (int t2 = 0; t2 < DT; ++t2) {
#pragma unroll
                for (int u = 0; u < 2; ++u) {
                    const f16x8 vf = Mfma<_Float16>::decode(vr[t2][2 * u], vr[t2][2 * u + 1]);
#pragma unroll
                    for (int nt = 0; nt < NQ; ++nt) o[nt][t2] = Mfma<_Float16>::run(vf, p[nt][u], o[nt][t2]);
                }
                __builtin_amdgcn_sched_barrier(0);
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
                        f32x4 x = Mfma<_Float16>::run(Mfma<_Float16>::decode(w[0], w[1]), p[nt][0], f32x4{0.f, 0.f, 0.f, 0.f});
                        x = Mfma<_Float16>::run(Mfma<_Float16>::decode(w[2], w[3]), p[nt][1], x);
                        if (t * 64 + tok <= last[nt]) o[nt][t2] += x;
                    }
                }
            }
        }
        if (more) load_v(t + 4, now.v);
    };
    // (kept in order: left to itself the scheduler decodes a whole tile ahead and spills)
    for (; t < t_hi && (t + 1) * 64 <= partly; t += 4) step(std::false_type());
    for (; t < t_hi; t += 4) step(std::true_type());

    // join the four waves
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
        if (nt > 0) __syncthreads();   // (before the first, all waves are done with the queries)
#pragma unroll
        for (int t2 = 0; t2 < DT; ++t2) {
            f32x4 x = o[nt][t2];
#pragma unroll
            for (int j = 0; j < 4; ++j) x[j] *= f;
            *reinterpret_cast<f32x4 *>(&sm.o[wave][m * LROW + 16 * t2 + 4 * g]) = x;
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
            for (int w = 0; w < 4; ++w) x += *reinterpret_cast<const f32x4 *>(&sm.o[w][row * LROW + ch]);
            if (a.n_splits > 1) {
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
        if (a.n_splits > 1 && (threadIdx.x & 15) == 0) {
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
        int lo = 0, hi = a.batch - 1;
        while (lo < hi) {
            const int mid = (lo + hi + 1) >> 1;
            if (a.cu[mid] <= tok) lo = mid;
            else hi = mid - 1;
        }
        b = lo;
        if (a.cu[b + 1] <= tok || a.cu[b] < 0 || a.cu[b + 1] > a.n_tokens) return;   // not rising: the first kernel left it out
    }
    const int len = a.lens[b] < 0 ? 0 : (a.lens[b] > PA_MAX_LEN ? PA_MAX_LEN : a.lens[b]);
    const int wanted = ((len + 63) / 64 + a.tiles_per_split - 1) / a.tiles_per_split;
    const int used = wanted < 1 ? 1 : (wanted > a.n_splits ? a.n_splits : wanted);
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

// Query rows per workgroup: as many 16-row tiles as a sequence has rows on average, up to 4.  Splits: enough
// workgroups to fill the chip, runs of at least 256 tokens (one tile per wave), at most 64 of them.
Plan paged_plan(int64_t n_tokens, int64_t batch, bool ragged, int n_heads, int n_kv_heads, int page, int64_t table_width)
{
    Plan p;
    const int64_t group = n_heads / n_kv_heads;
    const int64_t rows = ragged ? gq_cdiv(n_tokens * group, batch) : group;
    p.nq = rows <= 16 ? 1 : (rows <= 32 ? 2 : 4);
    const int mr = 16 * p.nq;
    p.n_items = ragged ? n_tokens * group / mr + batch : batch * gq_cdiv(group, mr);
    const int64_t tiles = gq_cdiv(table_width * page, 64), wgs = p.n_items * n_kv_heads;
    int64_t splits = gq_cdiv(2048, wgs);
    splits = std::min<int64_t>(splits, gq_cdiv(tiles, 4));
    splits = std::max<int64_t>(1, std::min<int64_t>(splits, PA_MAX_SPLITS));
    p.tiles_per_split = (int)std::max<int64_t>(4, gq_round_up(gq_cdiv(tiles, splits), 4));
    p.n_splits = (int)std::max<int64_t>(1, gq_cdiv(tiles, p.tiles_per_split));
    return p;
}

bool paged_sizes_ok(int64_t n_tokens, int64_t batch, int n_heads, int n_kv_heads, int head_dim, int page, int64_t table_width)
{
    return n_tokens >= 0 && n_tokens < ((int64_t)1 << 31) && batch >= 0 && batch < (1 << 24) && n_kv_heads > 0 && n_heads > 0 && n_heads <= 65536 &&
           n_heads % n_kv_heads == 0 && head_dim >= 16 && head_dim <= 128 && head_dim % 16 == 0 &&
           (page == 16 || page == 32 || page == 64 || page == 128) && table_width >= 0 && table_width * page < PA_MAX_LEN;
}

template <typename T>
int launch_paged(const PagedArgs &a, const Plan &p, hipStream_t s)
{
    const dim3 grid((unsigned)(p.n_items * a.n_kv_heads), (unsigned)p.n_splits);
#define GQ_PA(NC, NQ)                                                                                                   \
    do {                                                                                                                \
        if (a.page_log2 >= 6) hipLaunchKernelGGL((attention_paged_kernel<T, NC, NQ, true>), grid, dim3(256), 0, s, a);  \
        else hipLaunchKernelGGL((attention_paged_kernel<T, NC, NQ, false>), grid, dim3(256), 0, s, a);                  \
    } while (0)
    if (a.head_dim <= 64) {
        if (p.nq == 1) GQ_PA(1, 1);
        else if (p.nq == 2) GQ_PA(1, 2);
        else GQ_PA(1, 4);
    } else {
        if (p.nq == 1) GQ_PA(2, 1);
        else if (p.nq == 2) GQ_PA(2, 2);
        else GQ_PA(2, 4);
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

extern "C" int gq_attention_paged(void *out, int64_t out_token_stride, int64_t out_head_stride, const void *q, int64_t q_token_stride,
                                  int64_t q_head_stride, int dtype, int64_t n_tokens, int n_heads, const void *k_codes, const void *v_codes,
                                  const float *k_scale, const float *v_scale, int64_t n_pages, int n_kv_heads, int page, int head_dim,
                                  const int32_t *block_table, int64_t table_width, const int32_t *seq_lens, const int32_t *cu_seqlens,
                                  int64_t batch, float softmax_scale, void *workspace, size_t workspace_bytes, gq_stream_t stream)
{
    GQ_REQUIRE(dtype == GQ_F16 || dtype == GQ_BF16, "gq_attention_paged: dtype %d is neither fp16 (0) nor bf16 (1)", dtype);
    GQ_REQUIRE(paged_sizes_ok(n_tokens, batch, n_heads, n_kv_heads, head_dim, page, table_width) && n_pages >= 0,
               "gq_attention_paged: %d heads on %d, head_dim %d (a multiple of 16 up to 128), pages of %d (16, 32, 64 or 128): not supported", n_heads,
               n_kv_heads, head_dim, page);
    GQ_REQUIRE(cu_seqlens || n_tokens == batch, "gq_attention_paged: %lld tokens for %lld sequences need cu_seqlens", (long long)n_tokens,
               (long long)batch);
    GQ_REQUIRE(softmax_scale > 0.f && softmax_scale < INFINITY, "gq_attention_paged: the softmax scale must be positive and finite");
    if (n_tokens == 0 || batch == 0) return GQ_OK;
    GQ_REQUIRE(out && q && seq_lens && (table_width == 0 || block_table) && k_codes && v_codes && k_scale && v_scale,
               "gq_attention_paged: NULL pointer");
    GQ_REQUIRE(q_token_stride % 8 == 0 && q_head_stride % 8 == 0 && out_token_stride % 8 == 0 && out_head_stride % 8 == 0,
               "gq_attention_paged: strides must be multiples of 8 elements");
    GQ_REQUIRE((((uintptr_t)out | (uintptr_t)q | (uintptr_t)k_codes | (uintptr_t)v_codes | (uintptr_t)workspace) & 15) == 0,
               "gq_attention_paged: pointers must be 16-byte aligned");
    const Plan p = paged_plan(n_tokens, batch, cu_seqlens != nullptr, n_heads, n_kv_heads, page, table_width);
    GQ_REQUIRE(n_pages > 0, "gq_attention_paged: a cache without pages");
    GQ_REQUIRE(n_pages < ((int64_t)1 << 31) && p.n_items * n_kv_heads < ((int64_t)1 << 31) && n_tokens * n_heads < ((int64_t)1 << 31), "gq_attention_paged: too many query rows for one call");
    const size_t need = p.n_splits == 1 ? 0 : (size_t)n_tokens * n_heads * p.n_splits * (head_dim + 4) * sizeof(float);
    if (workspace_bytes < need || (need && !workspace)) {
        gq_set_error("gq_attention_paged: workspace of %zu bytes, %zu needed", workspace_bytes, need);
        return GQ_EWORKSPACE;
    }
    PagedArgs a;
    a.q = q, a.out = out, a.q_tok = q_token_stride, a.q_head = q_head_stride, a.o_tok = out_token_stride, a.o_head = out_head_stride;
    a.k_codes = (const uint8_t *)k_codes, a.v_codes = (const uint8_t *)v_codes, a.k_scale = k_scale, a.v_scale = v_scale;
    a.table = block_table, a.lens = seq_lens, a.cu = cu_seqlens;
    a.part_o = (float *)workspace;
    a.part_ml = (float *)workspace + (size_t)n_tokens * n_heads * p.n_splits * head_dim;
    a.n_tokens = n_tokens, a.n_pages = (int)n_pages, a.table_width = (int)table_width;
    a.batch = (int)batch, a.n_heads = n_heads, a.n_kv_heads = n_kv_heads, a.group = n_heads / n_kv_heads, a.head_dim = head_dim;
    a.page_log2 = __builtin_ctz((unsigned)page), a.tiles_per_split = p.tiles_per_split, a.n_splits = p.n_splits, a.n_items = (int)p.n_items;
    a.scale = softmax_scale * PA_LOG2E;
    return dtype == GQ_F16 ? launch_paged<_Float16>(a, p, (hipStream_t)stream) : launch_paged<__bf16>(a, p, (hipStream_t)stream);
}
