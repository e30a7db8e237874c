// Appending keys and values to a paged cache of 8-bit numbers, with the rotary embedding applied on the way.
//
// The cache holds e4m3 codes in pages of `page` tokens, one scale per (page, kv head) and tensor:
//   k_codes[n_pages][n_kv_heads][page][head_dim],  v_codes[n_pages][n_kv_heads][head_dim][page],  value = code * scale.
// Keys lie by token and values by channel because the attention over the cache reads both as operands of the matrix
// instruction whose inner index must be contiguous: channels for Q K^T, tokens for P V.
//
// Scales are powers of two, 2^e with the smallest e for which the page's largest finite magnitude a fits, a 2^-e <= 448.
// That costs an e4m3 number no precision (its error is relative), and it makes a page that fills up token by token
// well defined: when a new token needs a larger scale, the codes already there are re-expressed by a power of two,
// which only moves their exponent -- exact but for codes that become subnormal (below 2^-6 of a page whose largest code
// lies in (224, 448]).  Every value is rounded once from 32 bits: the rotated key never passes through 16 bits.
//
// One workgroup owns a (sequence's page, kv head, keys or values): it needs the largest magnitude before the first
// store, and nobody else may touch the page while codes are re-expressed.  The input stays in registers between the two.
// A thread takes 16 channels of each of two tokens of keys -- the two halves of 8 rotated pairs, one angle for both -- or 4
// tokens x 8 channels of values, whose codes go through LDS so that both the loads (by token) and the stores (by channel)
// are whole lines.  Rotary widths that are no multiple of 16 share a head out by the same 16 channels an item, see any_pairs.
// Bound by HBM for prompts (16-bit input in, one byte out), next to the vector instructions of rotation and rounding (74 %
// of the busy CUs' time): 4.2 TB/s, 111 us for 8 ragged prompts of 11314 tokens in all, 32 query heads on 32 of 128 channels,
// on operands that no cache holds; by a launch and dependent loads for single tokens (64 sequences: 6.7 us).
#include <type_traits>

#include "gq_common.h"

namespace {

constexpr float E4M3_MAX = 448.f;
constexpr int MIN_EXP = -100, MAX_EXP = 120;   // exponents of scales; MIN_EXP is a page of zeros

struct AppendArgs {
    const void *q, *k, *v;            // [n_tokens][heads][head_dim] by strides; q may be NULL
    void *q_out;
    int64_t q_tok, q_head, qo_tok, qo_head, k_tok, k_head, v_tok, v_head;   // strides in elements
    uint8_t *k_codes, *v_codes;
    float *k_scale, *v_scale;
    const float *cos_t, *sin_t;       // [max_pos][rot / 2]
    const int32_t *table, *past, *cu;   // cu NULL: one token per sequence
    int64_t n_tokens, max_pos, n_pages, table_width;
    int batch, n_heads, n_kv_heads, head_dim, page, rot, interleaved, n_items, q_parts;
};

template <typename T>
__device__ __forceinline__ void load8f(const T *p, float (&f)[8])
{
    const u32x4 raw = *reinterpret_cast<const u32x4 *>(p);
    T v[8];
    __builtin_memcpy(v, &raw, 16);
#pragma unroll
    for (int i = 0; i < 8; ++i) f[i] = static_cast<float>(v[i]);
}

template <typename T>
__device__ __forceinline__ void store8f(T *p, const float (&f)[8])
{
    T v[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = static_cast<T>(f[i]);
    u32x4 raw;
    __builtin_memcpy(&raw, v, 16);
    *reinterpret_cast<u32x4 *>(p) = raw;
}

// Pair p of a head: 16 channels as two runs of 8, at `lo` and `hi`.  Of a rotated part in two halves they are partners.
__device__ __forceinline__ void pair_channels(int p, int rot, int interleaved, int &lo, int &hi)
{
    const bool halves = !interleaved && 16 * p < rot;
    lo = halves ? 8 * p : 16 * p;
    hi = halves ? lo + (rot >> 1) : lo + 8;
}

// Loads pair p of a head and rotates it by the angles of cos_r / sin_r (rows of the tables; NULL: as it is), each product
// and the sum rounded in 32 bits.
template <typename T>
__device__ __forceinline__ void load_pair(const T *head, int p, const float *cos_r, const float *sin_r, int rot, int interleaved, float (&a)[8],
                                          float (&b)[8])
{
    int lo, hi;
    pair_channels(p, rot, interleaved, lo, hi);
    load8f(head + lo, a);
    load8f(head + hi, b);
    if (16 * p >= rot) return;
    // the 8 angles of this pair: of channels (lo + i, hi + i), or of (2 j, 2 j + 1) for j = 8 p + i
    float c[8], s[8];
    *reinterpret_cast<f32x4 *>(c) = *reinterpret_cast<const f32x4 *>(cos_r + 8 * p);
    *reinterpret_cast<f32x4 *>(c + 4) = *reinterpret_cast<const f32x4 *>(cos_r + 8 * p + 4);
    *reinterpret_cast<f32x4 *>(s) = *reinterpret_cast<const f32x4 *>(sin_r + 8 * p);
    *reinterpret_cast<f32x4 *>(s + 4) = *reinterpret_cast<const f32x4 *>(sin_r + 8 * p + 4);
    const auto turn = [](float &x, float &y, float cs, float sn) {
        const float u = x, v = y;
        x = __fsub_rn(__fmul_rn(u, cs), __fmul_rn(v, sn));
        y = __fadd_rn(__fmul_rn(v, cs), __fmul_rn(u, sn));
    };
    if (interleaved) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            turn(a[2 * i], a[2 * i + 1], c[i], s[i]);
            turn(b[2 * i], b[2 * i + 1], c[4 + i], s[4 + i]);
        }
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) turn(a[i], b[i], c[i], s[i]);
    }
}

// Any other even rotary width (a kernel of its own: the pairs' second sides are at no aligned place then).  Item p of a head
// takes r = half - 8 p (0 to 8) of the pairs (8 p + i, 8 p + i + half); where pairs end inside its 16 channels the places
// left take channels that are not rotated, so that the items share the head out among them:
//   a_i: channel 8 p + i where i < r, else 16 p + 8 + i;   b_i: channel (r > 0 ? 8 p + half : 16 p) + i
// (half = 8 P + r for the item P where pairs end: its b goes on into the channels from 2 half = 16 P + 2 r on, its a takes
// the last 8 - r before 16 P + 16).  Of interleaved pairs a and b are the item's two runs of 8.  The second sides are loaded
// and stored at the alignment of an element, which the memory unit takes.  Single tokens take the launch's time as ever; 8
// ragged prompts of 11314 tokens of 32/32 heads of 80 (cached operands): 119 us at a width of 40, 92 at 32 and at 48
// (interleaved 106), of 128 channels 164 at 72, 111 at 64.
__device__ __forceinline__ int any_pairs(int p, int half)
{
    const int r = half - 8 * p;
    return r < 0 ? 0 : (r > 8 ? 8 : r);
}

struct AnyPlaces {
    int r, split, a, b;   // pairs; elements of a that lie at 8 p, where the rest of it and b lie
};

__device__ __forceinline__ AnyPlaces any_places(int p, int half, int interleaved)
{
    const int r = any_pairs(p, half);
    if (interleaved) return {r, 0, 16 * p, 16 * p + 8};
    return {r, r, 16 * p + 8, r > 0 ? 8 * p + half : 16 * p};
}

template <typename T>
__device__ __forceinline__ void load8f_any(const T *p, float (&f)[8])
{
    T v[8];
    __builtin_memcpy(v, p, sizeof(v));
#pragma unroll
    for (int i = 0; i < 8; ++i) f[i] = static_cast<float>(v[i]);
}

template <typename T>
__device__ __forceinline__ void load_pair_any(const T *head, int p, const float *cos_r, const float *sin_r, int half, int interleaved, bool last_row,
                                              float (&a)[8], float (&b)[8])
{
    const AnyPlaces at = any_places(p, half, interleaved);
    if (at.split < 8) load8f(head + at.a, a);
    if (at.split > 0) {
        float x[8];
        load8f(head + 8 * p, x);
#pragma unroll
        for (int i = 0; i < 8; ++i) a[i] = i < at.split ? x[i] : a[i];
    }
    load8f_any(head + at.b, b);
    if (at.r == 0) return;
    float c[8], s[8];
    if (at.r == 8 || !last_row) {   // (8 angles also where fewer are left: the next row's follow, but not behind the table's last)
        __builtin_memcpy(c, cos_r + 8 * p, sizeof(c));
        __builtin_memcpy(s, sin_r + 8 * p, sizeof(s));
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            c[i] = i < at.r ? cos_r[8 * p + i] : 0.f;
            s[i] = i < at.r ? sin_r[8 * p + i] : 0.f;
        }
    }
    const auto turn = [&](int i, float &x, float &y) {
        if (i >= at.r) return;
        const float u = x, v = y;
        x = __fsub_rn(__fmul_rn(u, c[i]), __fmul_rn(v, s[i]));
        y = __fadd_rn(__fmul_rn(v, c[i]), __fmul_rn(u, s[i]));
    };
    if (interleaved) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            turn(i, a[2 * i], a[2 * i + 1]);
            turn(4 + i, b[2 * i], b[2 * i + 1]);
        }
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) turn(i, a[i], b[i]);
    }
}

// 8 elements each for the places of a and b in a head's row
template <typename E>
__device__ __forceinline__ void store_pair_any(E *row, int p, int half, int interleaved, const E (&a)[8], const E (&b)[8])
{
    const AnyPlaces at = any_places(p, half, interleaved);
    if (at.split == 0) {
        __builtin_memcpy(row + at.a, a, sizeof(a));
    } else if (at.split == 8) {
        __builtin_memcpy(row + 8 * p, a, sizeof(a));
    } else {
        const auto pieces = [&](auto width) {
            constexpr int W = decltype(width)::value;
#pragma unroll
            for (int i = 0; i < 8; i += W) __builtin_memcpy(row + (i < at.split ? 8 * p : at.a) + i, a + i, W * sizeof(E));
        };
        if (at.split % 4 == 0) pieces(std::integral_constant<int, 4>());
        else if (at.split % 2 == 0) pieces(std::integral_constant<int, 2>());
        else pieces(std::integral_constant<int, 1>());
    }
    __builtin_memcpy(row + at.b, b, sizeof(b));
}

__device__ __forceinline__ unsigned to_codes4(float a, float b, float c, float d)
{
    // infinities saturate (the conversion would make them NaN); NaN stays NaN
    const auto sat = [](float x) { return x > E4M3_MAX ? E4M3_MAX : (x < -E4M3_MAX ? -E4M3_MAX : x); };
    int r = __builtin_amdgcn_cvt_pk_fp8_f32(sat(a), sat(b), 0, false);
    return (unsigned)__builtin_amdgcn_cvt_pk_fp8_f32(sat(c), sat(d), r, true);
}

__device__ __forceinline__ unsigned scale_codes4(unsigned w, float f)
{
    return to_codes4(__builtin_amdgcn_cvt_f32_fp8(w, 0) * f, __builtin_amdgcn_cvt_f32_fp8(w, 1) * f, __builtin_amdgcn_cvt_f32_fp8(w, 2) * f,
                     __builtin_amdgcn_cvt_f32_fp8(w, 3) * f);
}

__device__ __forceinline__ float pow2f(int e) { return __uint_as_float((unsigned)(e + 127) << 23); }

// the smallest e with a 2^-e <= 448 = 1.75 * 2^8, for the bits of a finite a >= 0
__device__ __forceinline__ int exponent_for(unsigned bits)
{
    const int e = (int)(bits >> 23) - 135 + ((bits & 0x7fffff) > 0x600000);
    return e < MIN_EXP ? MIN_EXP : (e > MAX_EXP ? MAX_EXP : e);
}

// The sequence that `pos` of a rising row of batch + 1 starts lies in: the last b < batch with f(b) <= pos (-1: none), one
// less than how many there are; a wave looks at 64 at a time.
template <typename F>
__device__ __forceinline__ int find_sequence(int batch, int64_t pos, F f)
{
    const int lane = threadIdx.x & 63;
    int n = 0;
    for (int b0 = 0; b0 < batch; b0 += 64) {
        const int c = __popcll(__ballot(b0 + lane < batch && f(b0 + lane) <= pos));
        n += c;
        if (c < 64) break;
    }
    return __builtin_amdgcn_readfirstlane(n) - 1;
}

// ANY: the rotary width is no multiple of 16
template <typename T, bool ANY>
__device__ __forceinline__ void append_page(const AppendArgs &a, int item, int head, bool is_v, unsigned *sm_max, unsigned *sm_tile)
{
    const int tid = threadIdx.x, nt = blockDim.x;
    int b = item, j = 0;
    int64_t row0 = item, n = 1;
    if (a.cu) {
        // sequence b starts at item cu[b] / page + 2 b: room for the (n + page - 2) / page + 1 pages it can touch
        const auto start = [&](int s) { return (int64_t)a.cu[s] / a.page + 2 * (int64_t)s; };
        b = find_sequence(a.batch, item, start);
        if (b < 0) return;
        j = (int)(item - start(b));
        row0 = a.cu[b];
        n = (int64_t)a.cu[b + 1] - row0;
        if (row0 < 0 || n <= 0 || row0 + n > a.n_tokens) return;
    }
    const int64_t past = a.past[b];
    if (past < 0) return;
    const int64_t pidx = past / a.page + j, first = pidx * a.page;   // the page's place in its sequence, its first position
    int64_t end = past + n;
    if (a.rot && end > a.max_pos) end = a.max_pos;   // positions without an angle are not stored
    const int s0 = (int)(past > first ? past - first : 0);
    const int s1 = (int)(end - first < a.page ? end - first : a.page);
    if (s1 <= s0 || pidx >= a.table_width) return;
    const int64_t page_id = a.table[(int64_t)b * a.table_width + pidx];
    if (page_id < 0 || page_id >= a.n_pages) return;

    const int d = a.head_dim;
    const T *x = is_v ? (const T *)a.v + head * a.v_head : (const T *)a.k + head * a.k_head;
    const int64_t tok_stride = is_v ? a.v_tok : a.k_tok;
    const int64_t block = page_id * a.n_kv_heads + head;
    uint8_t *codes = (is_v ? a.v_codes : a.k_codes) + block * a.page * d;
    float *scale = (is_v ? a.v_scale : a.k_scale) + block;
    const float old = *scale;
    const int64_t row_of_0 = row0 + first - past;   // row of the page's slot 0, were it new

    // Items of keys: a token and 16 channels, two for a thread.  Items of values: 4 tokens (of one word of codes) and 8
    // channels, one for a thread.
    float f[2][16];   // (f[t / 2][8 (t % 2) ..]: token t of the values)
    const int n_pairs = d >> 4, n_ch = d >> 3;
    const int n_keys = (s1 - s0) * n_pairs;
    const int quad0 = s0 >> 2, n_quads = ((s1 - 1) >> 2) - quad0 + 1, n_vals = n_quads * n_ch;
    const int quad = quad0 + tid / n_ch, ch = tid % n_ch;
    unsigned most = 0;
    const auto measure = [&](float v) {
        const unsigned bits = __float_as_uint(v) & 0x7fffffffu;
        if (bits < 0x7f800000u && bits > most) most = bits;
    };
    if (is_v) {
        if (tid < n_vals) {
#pragma unroll
            for (int t = 0; t < 4; ++t) {
                float (&g)[8] = *reinterpret_cast<float (*)[8]>(&f[t >> 1][8 * (t & 1)]);
                const int s = 4 * quad + t;
                if (s >= s0 && s < s1) {
                    load8f(x + (row_of_0 + s) * tok_stride + 8 * ch, g);
                } else {
#pragma unroll
                    for (int i = 0; i < 8; ++i) g[i] = 0.f;
                }
            }
#pragma unroll
            for (int k = 0; k < 32; ++k) measure(f[k >> 4][k & 15]);
        }
    } else {
#pragma unroll
        for (int k = 0; k < 2; ++k) {
            const int it = tid + k * nt;
            if (it < n_keys) {
                const int s = s0 + it / n_pairs;
                const int64_t at = (first + s) * (a.rot >> 1);
                float (&lo)[8] = *reinterpret_cast<float (*)[8]>(&f[k][0]), (&hi)[8] = *reinterpret_cast<float (*)[8]>(&f[k][8]);
                const T *row = x + (row_of_0 + s) * tok_stride;
                if constexpr (ANY) load_pair_any(row, it % n_pairs, a.cos_t + at, a.sin_t + at, a.rot >> 1, a.interleaved, first + s >= a.max_pos - 1, lo, hi);
                else load_pair(row, it % n_pairs, a.cos_t + at, a.sin_t + at, a.rot, a.interleaved, lo, hi);
#pragma unroll
                for (int i = 0; i < 16; ++i) measure(f[k][i]);
            }
        }
    }
#pragma unroll
    for (int off = 32; off > 0; off >>= 1) {
        const unsigned o = __shfl_xor(most, off, 64);
        most = o > most ? o : most;
    }
    if (nt > 64) {
        if ((tid & 63) == 0) sm_max[tid >> 6] = most;
        __syncthreads();
        for (int w = 0; w < nt >> 6; ++w) most = sm_max[w] > most ? sm_max[w] : most;
    }
    int e = exponent_for(most);
    if (s0 > 0) {
        // the tokens already there keep the scale from falling; a scale that is no power of two is rounded up to one, and one
        // that is no number leaves them NaN
        const unsigned ob = __float_as_uint(old);
        int eo = old > 0.f && old < INFINITY ? (int)(ob >> 23) - 127 + ((ob & 0x7fffff) != 0) : MIN_EXP;
        eo = eo < MIN_EXP ? MIN_EXP : (eo > MAX_EXP ? MAX_EXP : eo);
        e = eo > e ? eo : e;
        const float ratio = old > 0.f && old < INFINITY ? old * pow2f(-e) : (old <= 0.f ? 0.f : NAN);
        if (ratio != 1.f) {
            if (is_v) {
                const int words = (s0 + 3) >> 2;
                for (int i = tid; i < d * words; i += nt) {
                    const int row = i / words, w = i - row * words;
                    unsigned *p = reinterpret_cast<unsigned *>(codes + row * a.page) + w;
                    const unsigned was = *p;
                    const int kept = s0 - 4 * w;   // of the word's four tokens
                    const unsigned mask = kept >= 4 ? 0xffffffffu : ((1u << (8 * kept)) - 1);
                    *p = (scale_codes4(was, ratio) & mask) | (was & ~mask);
                }
            } else {
                for (int i = tid; i < s0 * (d >> 2); i += nt) {
                    unsigned *p = reinterpret_cast<unsigned *>(codes) + i;
                    *p = scale_codes4(*p, ratio);
                }
            }
            __syncthreads();   // a word of values may hold tokens of both kinds
        }
    }
    if (tid == 0) *scale = pow2f(e);
    const float inv = pow2f(-e);
    if (!is_v) {
#pragma unroll
        for (int k = 0; k < 2; ++k) {
            const int it = tid + k * nt;
            if (it < n_keys) {
                uint8_t *row = codes + (s0 + it / n_pairs) * d;
                const float (&g)[16] = f[k];
                const u32x2 wa = {to_codes4(g[0] * inv, g[1] * inv, g[2] * inv, g[3] * inv), to_codes4(g[4] * inv, g[5] * inv, g[6] * inv, g[7] * inv)};
                const u32x2 wb = {to_codes4(g[8] * inv, g[9] * inv, g[10] * inv, g[11] * inv), to_codes4(g[12] * inv, g[13] * inv, g[14] * inv, g[15] * inv)};
                if constexpr (ANY) {
                    uint8_t ca[8], cb[8];
                    __builtin_memcpy(ca, &wa, 8);
                    __builtin_memcpy(cb, &wb, 8);
                    store_pair_any(row, it % n_pairs, a.rot >> 1, a.interleaved, ca, cb);
                } else {
                    int lo, hi;
                    pair_channels(it % n_pairs, a.rot, a.interleaved, lo, hi);
                    *reinterpret_cast<u32x2 *>(row + lo) = wa;
                    *reinterpret_cast<u32x2 *>(row + hi) = wb;
                }
            }
        }
        return;
    }
    // A word of 4 tokens of channel c: in LDS at [c][word], the words of a row permuted by its 8 channels' number (16 lanes
    // with 16 such numbers write side by side); a word that is only partly new goes out by bytes.
    const int row_words = a.page >> 2;
    const auto put = [&](int c, int q, unsigned w) {
        uint8_t *p = codes + c * a.page + 4 * q;
        if (4 * q >= s0 && 4 * q + 4 <= s1) {
            *reinterpret_cast<unsigned *>(p) = w;
        } else {
#pragma unroll
            for (int t = 0; t < 4; ++t)
                if (4 * q + t >= s0 && 4 * q + t < s1) p[t] = (uint8_t)(w >> (8 * t));
        }
    };
    if (tid < n_vals) {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const unsigned w = to_codes4(f[0][i] * inv, f[0][8 + i] * inv, f[1][i] * inv, f[1][8 + i] * inv);
            if (n_quads == 1) put(8 * ch + i, quad, w);
            else sm_tile[(8 * ch + i) * row_words + (quad ^ (ch & (row_words - 1)))] = w;
        }
    }
    if (n_quads == 1) return;
    __syncthreads();
    const int pieces = a.page >> 4;   // of 16 tokens
    for (int i = tid; i < d * pieces; i += nt) {
        const int c = i / pieces, q = 4 * (i - c * pieces);
        u32x4 w;
#pragma unroll
        for (int k = 0; k < 4; ++k) w[k] = sm_tile[c * row_words + ((q + k) ^ ((c >> 3) & (row_words - 1)))];
        if (4 * q >= s0 && 4 * q + 16 <= s1) {
            *reinterpret_cast<u32x4 *>(codes + c * a.page + 4 * q) = w;
        } else {
#pragma unroll
            for (int k = 0; k < 4; ++k)
                if (4 * (q + k) < s1 && 4 * (q + k) + 4 > s0) put(c, q + k, w[k]);
        }
    }
}

// The query rows of a token, or part of its heads: a thread takes 16 channels, both sides of a rotated pair, so that q_out may be q.
template <typename T, bool ANY>
__device__ __forceinline__ void rotate_query(const AppendArgs &a, int64_t token, int part)
{
    int64_t pos;
    if (a.cu) {
        if (token < a.cu[0] || token >= a.cu[a.batch]) return;   // behind the last sequence: left as it is
        const int b = find_sequence(a.batch, token, [&](int s) { return (int64_t)a.cu[s]; });
        if (b < 0) return;
        pos = a.past[b] < 0 ? -1 : (int64_t)a.past[b] + (token - a.cu[b]);
    } else {
        pos = a.past[token];
    }
    const bool known = pos >= 0 && pos < a.max_pos;
    const int64_t angle = known ? pos : 0, at = angle * (a.rot >> 1);
    const int n_pairs = a.head_dim >> 4, n = a.n_heads * n_pairs;
    for (int i = part * blockDim.x + threadIdx.x; i < n; i += a.q_parts * blockDim.x) {
        const int head = i / n_pairs, p = i - head * n_pairs;
        float lo[8], hi[8];
        const T *x = (const T *)a.q + token * a.q_tok + head * a.q_head;
        if constexpr (ANY) load_pair_any(x, p, a.cos_t + at, a.sin_t + at, a.rot >> 1, a.interleaved, angle >= a.max_pos - 1, lo, hi);
        else load_pair(x, p, a.cos_t + at, a.sin_t + at, a.rot, a.interleaved, lo, hi);
        if (!known) {
#pragma unroll
            for (int k = 0; k < 8; ++k) lo[k] = hi[k] = NAN;
        }
        T *y = (T *)a.q_out + token * a.qo_tok + head * a.qo_head;
        if constexpr (ANY) {
            T ya[8], yb[8];
#pragma unroll
            for (int k = 0; k < 8; ++k) {
                ya[k] = static_cast<T>(lo[k]);
                yb[k] = static_cast<T>(hi[k]);
            }
            store_pair_any(y, p, a.rot >> 1, a.interleaved, ya, yb);
        } else {
            int cl, chh;
            pair_channels(p, a.rot, a.interleaved, cl, chh);
            store8f(y + cl, lo);
            store8f(y + chh, hi);
        }
    }
}

template <typename T, bool ANY>
__global__ __launch_bounds__(512) void kv_append_kernel(const AppendArgs a)
{
    __shared__ unsigned sm_max[8];
    extern __shared__ unsigned sm_tile[];   // values of a page, where whole words of tokens are new
    const unsigned n_kv = (unsigned)a.n_items * a.n_kv_heads * 2;
    if (blockIdx.x < n_kv) {
        const unsigned ih = blockIdx.x >> 1, item = ih / a.n_kv_heads;
        append_page<T, ANY>(a, (int)item, (int)(ih - item * a.n_kv_heads), blockIdx.x & 1, sm_max, sm_tile);
    } else {
        const unsigned i = blockIdx.x - n_kv, token = i / a.q_parts;
        rotate_query<T, ANY>(a, token, (int)(i - token * a.q_parts));
    }
}

}  // namespace

extern "C" int gq_kv_append(const gq_kv_append_args *args, gq_stream_t stream)
{
    GQ_REQUIRE(args, "gq_kv_append: NULL pointer");
    const gq_paged_cache cache = args->cache;
    const gq_rows k = args->k, v = args->v, q = args->q, q_out = args->q_out;
    const int64_t dtype = args->dtype, n_tokens = args->n_tokens, n_heads = args->n_heads, n_pages = cache.n_pages, n_kv_heads = cache.n_kv_heads;
    const int64_t page = cache.page, head_dim = cache.head_dim, table_width = args->table_width, batch = args->batch, max_pos = args->max_pos;
    const int64_t rotary_dim = args->rotary_dim;
    const int32_t *block_table = args->block_table, *past_lens = args->past_lens, *cu_seqlens = args->cu_seqlens;
    const float *cos_t = args->cos, *sin_t = args->sin;
    GQ_REQUIRE(dtype == GQ_F16 || dtype == GQ_BF16, "gq_kv_append: dtype %lld is neither fp16 (0) nor bf16 (1)", (long long)dtype);
    GQ_REQUIRE(head_dim >= 16 && head_dim <= 128 && head_dim % 16 == 0, "gq_kv_append: head_dim %lld is not a multiple of 16 up to 128",
               (long long)head_dim);
    GQ_REQUIRE(page == 16 || page == 32 || page == 64 || page == 128, "gq_kv_append: pages of %lld tokens: 16, 32, 64 or 128 are supported",
               (long long)page);
    GQ_REQUIRE(n_kv_heads > 0 && n_pages >= 0 && n_tokens >= 0 && batch >= 0 && table_width >= 0, "gq_kv_append: negative size");
    GQ_REQUIRE(batch < (1 << 24) && n_tokens < ((int64_t)1 << 31) && n_kv_heads <= 65536 && n_heads <= 65536, "gq_kv_append: too many tokens, sequences or heads");
    GQ_REQUIRE(cu_seqlens || n_tokens == batch, "gq_kv_append: %lld tokens for %lld sequences need cu_seqlens", (long long)n_tokens, (long long)batch);
    GQ_REQUIRE(rotary_dim == 0 || (rotary_dim >= 16 && rotary_dim <= head_dim && rotary_dim % 2 == 0),
               "gq_kv_append: rotary_dim %lld is neither 0 nor an even number from 16 to head_dim", (long long)rotary_dim);
    const bool any = rotary_dim % 16 != 0;
    if (n_tokens == 0 || batch == 0) return GQ_OK;
    GQ_REQUIRE(cache.k_codes && cache.v_codes && cache.k_scale && cache.v_scale && k.data && v.data && block_table && past_lens, "gq_kv_append: NULL pointer");
    GQ_REQUIRE(!rotary_dim || (cos_t && sin_t && max_pos > 0), "gq_kv_append: a rotation needs the tables of cosines and sines");
    GQ_REQUIRE(!q.data || (q_out.data && n_heads > 0 && rotary_dim), "gq_kv_append: q needs an output, heads and a rotation");
    GQ_REQUIRE(k.token_stride % 8 == 0 && k.head_stride % 8 == 0 && v.token_stride % 8 == 0 && v.head_stride % 8 == 0 &&
                   (!q.data || (q.token_stride % 8 == 0 && q.head_stride % 8 == 0 && q_out.token_stride % 8 == 0 && q_out.head_stride % 8 == 0)),
               "gq_kv_append: strides must be multiples of 8 elements");
    GQ_REQUIRE(!q.data || gq_rows_apart(q_out, n_tokens, n_heads, head_dim), "gq_kv_append: rows of q_out overlap");
    GQ_REQUIRE((((uintptr_t)cache.k_codes | (uintptr_t)cache.v_codes | (uintptr_t)k.data | (uintptr_t)v.data | (uintptr_t)q.data | (uintptr_t)q_out.data) & 15) == 0 &&
                   (((uintptr_t)cos_t | (uintptr_t)sin_t) & (any ? 3 : 15)) == 0,
               "gq_kv_append: pointers must be 16-byte aligned (the tables' 4 where rotary_dim is no multiple of 16)");
    AppendArgs a;
    a.q = q.data, a.k = k.data, a.v = v.data, a.q_out = q_out.data;
    a.q_tok = q.token_stride, a.q_head = q.head_stride, a.qo_tok = q_out.token_stride, a.qo_head = q_out.head_stride;
    a.k_tok = k.token_stride, a.k_head = k.head_stride, a.v_tok = v.token_stride, a.v_head = v.head_stride;
    a.k_codes = (uint8_t *)cache.k_codes, a.v_codes = (uint8_t *)cache.v_codes, a.k_scale = cache.k_scale, a.v_scale = cache.v_scale;
    a.cos_t = cos_t, a.sin_t = sin_t, a.table = block_table, a.past = past_lens, a.cu = cu_seqlens;
    a.n_tokens = n_tokens, a.max_pos = max_pos, a.n_pages = n_pages, a.table_width = table_width;
    a.batch = (int)batch, a.n_heads = (int)n_heads, a.n_kv_heads = (int)n_kv_heads, a.head_dim = (int)head_dim, a.page = (int)page;
    a.rot = (int)rotary_dim, a.interleaved = args->interleaved != 0;
    const int64_t n_items = cu_seqlens ? n_tokens / page + 2 * batch : batch;
    // Two 16-channel items of keys for each thread of a page, which is one 4 x 8 item of values; one wave for single tokens.
    // Queries: an item for each thread where tokens are few, a workgroup for a token where they fill the chip.
    const int64_t pairs = (cu_seqlens ? page : 1) * (head_dim / 16);
    const int threads = pairs <= 128 ? 64 : (pairs <= 256 ? 128 : (pairs <= 512 ? 256 : 512));
    a.q_parts = n_tokens < 1024 ? (int)gq_cdiv(n_heads * (head_dim / 16), threads) : 1;
    const int64_t q_blocks = q.data ? n_tokens * a.q_parts : 0;
    const size_t lds = cu_seqlens ? (size_t)(page * head_dim) : 0;
    const int64_t grid = n_items * n_kv_heads * 2 + q_blocks;
    GQ_REQUIRE(grid < GQ_MAX_THREADS / threads, "gq_kv_append: too many tokens for one call");
    a.n_items = (int)n_items;
#define GQ_KA(T, ANY) hipLaunchKernelGGL((kv_append_kernel<T, ANY>), dim3((unsigned)grid), dim3(threads), lds, (hipStream_t)stream, a)
    if (dtype == GQ_F16) {
        if (any) GQ_KA(_Float16, true);
        else GQ_KA(_Float16, false);
    } else {
        if (any) GQ_KA(__bf16, true);
        else GQ_KA(__bf16, false);
    }
#undef GQ_KA
    GQ_LAUNCH_CHECK();
    return GQ_OK;
}
