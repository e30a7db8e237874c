// Attention over whole prompts: packed sequences of different lengths, grouped heads, causal or not.
//
//   S = scale Q K^T (masked),  m = row max,  P = e^(S - m),  O = P V / sum P
// in one pass over the keys: a running (m, l, O) per query row, O and l rescaled when m grows.
//
// A workgroup of 4 waves takes 128 query rows of one head, a wave 32 of them, 64 keys at a time.  Everything is
// computed transposed, S^T = K Q^T and O^T = V^T P^T with 32 x 32 x 16 matrix instructions: a lane then holds, of its
// query row (its column), tokens 8 i + 4 h + 0..3 of the keys (h = lane / 32), and that is what it supplies as the
// operand P^T when the inner index is taken in that order -- the weights go from the first product to the second
// without leaving their lane, the row's maximum needs one exchange between two lanes.  K and V tiles are copied to LDS
// by the asynchronous copy, 16-byte chunks permuted within a row (by the row) so that both the row-wise reads of K and
// the transposing reads of V (4 tokens x 16 channels per 16 lanes) touch all banks.
// Rows behind a sequence's end and channels behind head_dim are out of the buffer descriptor's range and arrive as 0.
//
// Bound by the matrix core next to the softmax's vector instructions: 4 head_dim flops per visible (query, key) pair and
// one exponential; for sequences of a few thousand tokens also by a workgroup's queries and outputs (64 KB at 128 channels,
// which the other workgroup of a CU has to hide).  Measured with 128 channels, causal, on operands that no cache holds:
// 16384 tokens of 32/8 heads 1940 us (1133 TFLOP/s, 0.9 of what a library product of 8192^3 reaches), 4 x 2048 tokens of
// 32 heads 176 us (783 TFLOP/s, 1.5 TB/s: of the busy CUs' time the matrix pipe takes 47 %, the vector unit 52 %), packed
// sequences of 1 to 3001 tokens 323 to 340 us (830 TFLOP/s), 77 tokens 6.5 us (a launch).
#include <type_traits>

#include "gq_common.h"

namespace {

constexpr float AP_LOG2E = 1.44269504088896340736f;
constexpr int AP_Q = 128, AP_K = 64;
constexpr unsigned AP_OUT_OF_RANGE = 0x80000000u;

struct PromptArgs {
    const void *q, *k, *v;
    void *out;
    int64_t q_tok, q_head, k_tok, k_head, v_tok, v_head, o_tok, o_head;   // strides in elements
    const int32_t *cu;   // NULL: one sequence
    int64_t n_tokens;
    int batch, n_heads, group, head_dim, n_items, causal;
    float scale;         // softmax scale * log2 e
};

typedef __amdgpu_buffer_rsrc_t ap_rsrc_t;

template <typename T> struct Mma;
template <> struct Mma<_Float16> {
    typedef f16x8 vec;
    static constexpr unsigned EXPONENT_ONE = 0x04000400u;
    static constexpr float LIFT = 7.f;
    static __device__ __forceinline__ f32x16 run(f16x8 a, f16x8 b, f32x16 c) { return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0); }
};
template <> struct Mma<__bf16> {
    typedef bf16x8 vec;
    static constexpr unsigned EXPONENT_ONE = 0x00800080u;
    static constexpr float LIFT = 0.f;
    static __device__ __forceinline__ f32x16 run(bf16x8 a, bf16x8 b, f32x16 c) { return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0); }
};

// Chunk c (of 16 bytes) of a row lies in place c ^ swizzle(row).  The banks take 256 bytes at a time: 16 lanes that read
// one chunk each of 16 adjacent rows of K, 32 lanes that read 64 bytes each of 4 adjacent rows of V (measured: with
// c ^ (row & 7) the former run at half, the latter at a quarter of the rate).  256 bytes are 1 row of 16 chunks, 2 of 8,
// and rows of 12 begin in 4 different quarters, so the low bits of the row choose the quarter, the next the chunk in it.
template <int DP>
__device__ __forceinline__ int ap_swizzle(int row)
{
    return DP == 128 ? ((row & 3) << 2) | ((row >> 2) & 3) : (DP == 96 ? (row >> 2) & 3 : ((row & 2) << 1) | ((row >> 2) & 3));
}

// 3 workgroups to a CU where the registers allow it (up to 64 channels: 4 x 2048 tokens of 32/8 heads 110 -> 102 us, 8192
// tokens not causal 584 -> 567, on cached operands), else 2.
template <typename T, int DP>
__global__ __launch_bounds__(256, DP == 64 ? 3 : 2) void attention_prompt_kernel(const PromptArgs a)
{
    typedef typename Mma<T>::vec vec;
    constexpr int NCH = DP / 8;                       // 16-byte chunks of a row
    constexpr int PIECES = AP_K * NCH / 256;          // copy instructions per wave and tile
    constexpr int STEPS = DP / 16, DT = DP / 32;
    // Four objects, so that the compiler's own waits tell the copies into one from those into the next: of one object it
    // makes the reads of a tile wait for the copies of the tile after it.
    __shared__ __attribute__((aligned(1024))) T sm_k0[AP_K * DP], sm_k1[AP_K * DP], sm_v0[AP_K * DP], sm_v1[AP_K * DP];

    const int tid = threadIdx.x, lane = tid & 63, col = lane & 31, h = lane >> 5;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);   // uniform, so that what follows from it is scalar
    // workgroups of one head group run on one XCD (consecutive blocks go round the 8) and share its L2; long tiles first
    int head, item;
    if ((a.n_heads & 7) == 0) {
        const int per = a.n_heads >> 3, x = blockIdx.x & 7, i = blockIdx.x >> 3;
        head = x * per + i % per;
        item = i / per;
    } else {
        head = blockIdx.x % a.n_heads;
        item = blockIdx.x / a.n_heads;
    }
    item = a.n_items - 1 - item;
    int64_t row0 = 0, n = a.n_tokens;
    int tile = item;
    if (a.cu) {
        // Sequence b's tiles start at item cu[b] / 128 + b: room for all of them without the host knowing the lengths.
        // The starts rise, so b is one less than the number of starts up to this item; 64 are looked at at a time.
        // (The two starts that count are nearly always among those in the lanes.)
        int lo = -1, c = 0, mine = 0;
        for (int b0 = 0; b0 < a.batch; b0 += 64) {
            const int at = b0 + lane < a.batch ? b0 + lane : a.batch;
            mine = a.cu[at];
            c = __popcll(__ballot(b0 + lane < a.batch && mine / AP_Q + at <= item));
            lo += c;
            if (c < 64) break;
        }
        if (lo < 0) return;
        lo = __builtin_amdgcn_readfirstlane(lo);
        c = __builtin_amdgcn_readfirstlane(c);
        const bool here = c > 0 && c < 64;
        row0 = here ? __builtin_amdgcn_readlane(mine, c - 1) : a.cu[lo];
        n = (here ? __builtin_amdgcn_readlane(mine, c) : a.cu[lo + 1]) - row0;
        const int64_t t = item - (row0 / AP_Q + lo);
        if (row0 < 0 || n <= 0 || row0 + n > a.n_tokens || t < 0 || t * AP_Q >= n) return;
        tile = (int)t;
    }
    const int len = (int)n, q0 = tile * AP_Q;
    const int d = a.head_dim, head_kv = head / a.group;
    const int row = q0 + wave * 32 + col;            // this lane's query row in its sequence

    // what each lane copies of a tile: chunk `tid + 256 j` of the tile in LDS, from its row and unswizzled channel
    const unsigned k_row = (unsigned)(a.k_tok * sizeof(T)), v_row = (unsigned)(a.v_tok * sizeof(T));
    unsigned k_off[PIECES], v_off[PIECES];
#pragma unroll
    for (int j = 0; j < PIECES; ++j) {
        const int i = tid + 256 * j, r = i / NCH, c = (i - r * NCH) ^ ap_swizzle<DP>(r);
        k_off[j] = 8 * c < d ? r * k_row + 16 * c : AP_OUT_OF_RANGE;
        v_off[j] = 8 * c < d ? r * v_row + 16 * c : AP_OUT_OF_RANGE;
    }
    const T *kb = (const T *)a.k + row0 * a.k_tok + head_kv * a.k_head, *vb = (const T *)a.v + row0 * a.v_tok + head_kv * a.v_head;
    const auto stage = [&](int j, T *to_k, T *to_v) {
        const int rows = len - j * AP_K < AP_K ? len - j * AP_K : AP_K;
        const ap_rsrc_t rk = __builtin_amdgcn_make_buffer_rsrc((void *)(kb + (int64_t)j * AP_K * a.k_tok), 0, (int)((rows - 1) * k_row + 2 * d), 0x00020000);
        const ap_rsrc_t rv = __builtin_amdgcn_make_buffer_rsrc((void *)(vb + (int64_t)j * AP_K * a.v_tok), 0, (int)((rows - 1) * v_row + 2 * d), 0x00020000);
#pragma unroll
        for (int p = 0; p < PIECES; ++p)
            __builtin_amdgcn_raw_ptr_buffer_load_lds(rk, GQ_LDS_PTR(void, to_k + (wave * 64 + 256 * p) * 8), 16, (int)k_off[p], 0, 0, 0);
#pragma unroll
        for (int p = 0; p < PIECES; ++p)
            __builtin_amdgcn_raw_ptr_buffer_load_lds(rv, GQ_LDS_PTR(void, to_v + (wave * 64 + 256 * p) * 8), 16, (int)v_off[p], 0, 0, 0);
    };
    // all copies under way have arrived, everybody's (a barrier alone does not wait for the copies)
    const auto arrived = [] {
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        __syncthreads();
    };

    stage(0, sm_k0, sm_v0);
    vec qf[STEPS];
    {
        const T *qp = (const T *)a.q + (row0 + (row < len ? row : 0)) * a.q_tok + head * a.q_head;
#pragma unroll
        for (int s = 0; s < STEPS; ++s) {
            u32x4 raw = {0, 0, 0, 0};
            if (row < len && 16 * s + 8 * h < d) raw = *reinterpret_cast<const u32x4 *>(qp + 16 * s + 8 * h);
            __builtin_memcpy(&qf[s], &raw, 16);
        }
    }

    f32x16 o[DT];
#pragma unroll
    for (int t = 0; t < DT; ++t)
#pragma unroll
        for (int r = 0; r < 16; ++r) o[t][r] = 0.f;
    float mx = -INFINITY, l = 0.f;
    const int q_last = q0 + AP_Q - 1 < len - 1 ? q0 + AP_Q - 1 : len - 1;
    const int n_tiles = ((a.causal ? q_last : len - 1) + AP_K) / AP_K;
    // This wave's rows all see the first my_clear tiles, and of the tile after them the first `blocks` blocks of 32 tokens,
    // the last of those only in part.  (Tiles and waves begin at multiples of 32: the diagonal passes through one block.
    // Tokens behind the sequence are behind all its rows.)
    const int first_row = q0 + wave * 32;
    const int my_clear = first_row < len ? (a.causal ? first_row + 1 : len) / AP_K : 0;
    const int blocks = first_row < len ? ((a.causal ? first_row + 32 : len) - my_clear * AP_K + 31) / 32 : 0;
    const int see = a.causal ? row : len - 1;   // the last key this row sees

    // `tail`: of the tile only the first `blocks` (1 or 2) blocks of 32 tokens are visible, the last of them not to every
    // row unless the tile is clear to this wave.
    const auto compute = [&](auto tail, int j, const T *tk, const T *tv) {
        int lane = tid & 63;
        if constexpr (tail) asm volatile("" : "+v"(lane));   // (for a few tiles no addresses are kept in registers)
        const int col = lane & 31, h = lane >> 5;
        const int n_blocks = !tail || j < my_clear ? 2 : blocks, cut = !tail || j < my_clear ? 2 : blocks - 1;
        f32x16 s[2];
#pragma unroll
        for (int tb = 0; tb < 2; ++tb) {
#pragma unroll
            for (int r = 0; r < 16; ++r) s[tb][r] = 0.f;
            if (tb < n_blocks) {
                const int kr = 32 * tb + col, sw = ap_swizzle<DP>(kr);
#pragma unroll
                for (int st = 0; st < STEPS; ++st) {
                    const vec kf = *reinterpret_cast<const vec *>(tk + kr * DP + ((2 * st + h) ^ sw) * 8);
                    s[tb] = Mma<T>::run(kf, qf[st], s[tb]);
                }
            }
            if (tb >= cut) {
                const int rel = tb > cut ? -1 : see - (j * AP_K + 32 * tb) - 4 * h;
#pragma unroll
                for (int r = 0; r < 16; ++r)
                    if (8 * (r >> 2) + (r & 3) > rel) s[tb][r] = -INFINITY;
            }
        }
        float top = s[0][0];
#pragma unroll
        for (int tb = 0; tb < 2; ++tb)
#pragma unroll
            for (int r = 0; r < 16; ++r) top = fmaxf(top, s[tb][r]);
        top = gq_max_xor32(top) * a.scale;
        // The weights are 2^(s - mx + LIFT) for an mx that follows the row's maximum only when that is more than 8 above it:
        // O is rescaled once or twice a row instead of in most tiles (one of the wave's 32 rows finds a new maximum in nearly
        // every tile; 4 x 2048 tokens 183.5 -> 175.5 us).  They meet the values in the values' type, the matrix instruction's one
        // type for both, rounded once (11 bits in fp16, 8 in bf16); l sums them unrounded.  fp16 has 11 bits down to 2^-14 and
        // steps of 2^-24 below: LIFT = 7 uses the range up to 2^15 (of 65504), so that a weight 2^-21 of the row's largest
        // keeps its bits and what falls below half a step is 2^-32 of it, nothing even a million times over.
        if (__any(top > mx + 8.f)) {
            const float to = fmaxf(top, mx);
            const float f = mx == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(mx - to);
            mx = to;
            l *= f;
#pragma unroll
            for (int t = 0; t < DT; ++t)
#pragma unroll
                for (int r = 0; r < 16; ++r) o[t][r] *= f;
        }
        const float ref = mx == -INFINITY ? 0.f : mx - Mma<T>::LIFT;
        vec p[4];
#pragma unroll
        for (int tb = 0; tb < 2; ++tb)
#pragma unroll
            for (int r = 0; r < 16; ++r) {
                const float w = __builtin_amdgcn_exp2f(fmaf(s[tb][r], a.scale, -ref));
                l += w;
                p[2 * tb + (r >> 3)][r & 7] = static_cast<T>(w);
            }
        // V^T of channels 32 t .. and tokens 16 s2 + 4 h + 0..3, 16 s2 + 8 + 4 h + 0..3, as the weights have them
        const auto read_v = [&](int t, int s2) {
            vec vf;
#pragma unroll
            for (int half = 0; half < 2; ++half) {
                const int vr = 16 * s2 + 8 * half + 4 * h + ((lane >> 2) & 3), c0 = 32 * t + 16 * ((lane >> 4) & 1) + 4 * (lane & 3);
                const T *p0 = tv + vr * DP + (((c0 >> 3) ^ ap_swizzle<DP>(vr)) << 3) + (c0 & 7);
                const s16x4 x = __builtin_amdgcn_ds_read_tr16_b64_v4i16(GQ_LDS_PTR(s16x4, p0));
                __builtin_memcpy((char *)&vf + 8 * half, &x, 8);
            }
            return vf;
        };
        if constexpr (!tail) {
#pragma unroll
            for (int t = 0; t < DT; ++t)
#pragma unroll
                for (int s2 = 0; s2 < 4; ++s2) o[t] = Mma<T>::run(read_v(t, s2), p[s2], o[t]);
        } else {
#pragma unroll
            for (int tb = 0; tb < 2; ++tb) {
                if (tb >= n_blocks) break;
                if (tb != cut) {
#pragma unroll
                    for (int t = 0; t < DT; ++t)
#pragma unroll
                        for (int s2 = 2 * tb; s2 < 2 * tb + 2; ++s2) o[t] = Mma<T>::run(read_v(t, s2), p[s2], o[t]);
                    continue;
                }
                // 0 * inf and 0 * NaN are NaN: an infinity or NaN among these values must not reach the rows before it.
                // Adding one to an exponent field of all ones carries into the sign's place.
#pragma unroll
                for (int t = 0; t < DT; ++t) {
                    vec vf[2];
                    unsigned found = 0;
#pragma unroll
                    for (int i = 0; i < 2; ++i) {
                        vf[i] = read_v(t, 2 * tb + i);
                        unsigned x[4];
                        __builtin_memcpy(x, &vf[i], 16);
#pragma unroll
                        for (int w = 0; w < 4; ++w) found |= (x[w] & 0x7fff7fffu) + Mma<T>::EXPONENT_ONE;
                    }
                    if (!__any((found & 0x80008000u) != 0)) {
#pragma unroll
                        for (int i = 0; i < 2; ++i) o[t] = Mma<T>::run(vf[i], p[2 * tb + i], o[t]);
                        continue;
                    }
                    // one token at a time, added only to the rows that see it
#pragma unroll
                    for (int i = 0; i < 2; ++i)
#pragma unroll 1
                        for (int tok = 0; tok < 16; ++tok) {
                            vec one = vf[i];
#pragma unroll
                            for (int e = 0; e < 8; ++e)
                                if (8 * (e >> 2) + 4 * h + (e & 3) != tok) one[e] = static_cast<T>(0.f);
                            f32x16 x;
#pragma unroll
                            for (int r = 0; r < 16; ++r) x[r] = 0.f;
                            x = Mma<T>::run(one, p[2 * tb + i], x);
                            if (j * AP_K + 32 * tb + 16 * i + tok <= see) {
#pragma unroll
                                for (int r = 0; r < 16; ++r) o[t][r] += x[r];
                            }
                        }
                }
            }
        }
    };

    // pairs of tiles that are visible to the whole workgroup, then those that may be cut, each wave as far as it sees
    const int n_clear = (a.causal ? (q0 + 1) / AP_K : len / AP_K) & ~1;
    const int my_tiles = my_clear + (blocks > 0);
    int j = 0;
    for (; j < n_clear; j += 2) {
        arrived();
        stage(j + 1, sm_k1, sm_v1);
        compute(std::false_type(), j, sm_k0, sm_v0);
        arrived();
        if (j + 2 < n_tiles) stage(j + 2, sm_k0, sm_v0);
        compute(std::false_type(), j + 1, sm_k1, sm_v1);
    }
    for (; j < n_tiles; j += 2) {
        arrived();
        if (j + 1 < n_tiles) stage(j + 1, sm_k1, sm_v1);
        if (j < my_tiles) compute(std::true_type(), j, sm_k0, sm_v0);
        if (j + 1 >= n_tiles) break;
        arrived();
        if (j + 2 < n_tiles) stage(j + 2, sm_k0, sm_v0);
        if (j + 1 < my_tiles) compute(std::true_type(), j + 1, sm_k1, sm_v1);
    }

    l += __shfl_xor(l, 32, 64);
    const float inv = 1.f / l;
    // A lane holds 4 adjacent channels here and there of its row: through LDS (the wave's 32 rows, places as in the tiles),
    // so that rows are written in whole lines.  Two waves' rows fill a buffer of keys.
    constexpr int OUT = 32 * DP;
    static_assert(2 * OUT <= AP_K * DP && AP_Q == 4 * 32, "the rows of four waves fit the two buffers of keys");
    __syncthreads();
    T *so = (wave < 2 ? sm_k0 : sm_k1) + (wave & 1) * OUT;
#pragma unroll
    for (int t = 0; t < DT; ++t)
#pragma unroll
        for (int r4 = 0; r4 < 4; ++r4) {
            T y[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) y[i] = static_cast<T>(o[t][4 * r4 + i] * inv);
            u32x2 raw;
            __builtin_memcpy(&raw, y, 8);
            *reinterpret_cast<u32x2 *>(so + col * DP + (((4 * t + r4) ^ ap_swizzle<DP>(col)) << 3) + 4 * h) = raw;
        }
    __builtin_amdgcn_wave_barrier();
#pragma unroll
    for (int i = 0; i < DP / 16; ++i) {
        const int piece = i * 64 + lane, r = piece / NCH, c = piece - r * NCH;
        const int out_row = q0 + wave * 32 + r;
        const u32x4 x = *reinterpret_cast<const u32x4 *>(so + r * DP + ((c ^ ap_swizzle<DP>(r)) << 3));
        if (out_row < len && 8 * c < d) *reinterpret_cast<u32x4 *>((T *)a.out + (row0 + out_row) * a.o_tok + head * a.o_head + 8 * c) = x;
    }
}

template <typename T>
int launch_prompt(const PromptArgs &a, hipStream_t s)
{
    const dim3 grid((unsigned)a.n_items * (unsigned)a.n_heads);
#define GQ_AP(DP) hipLaunchKernelGGL((attention_prompt_kernel<T, DP>), grid, dim3(256), 0, s, a)
    if (a.head_dim <= 64) GQ_AP(64);
    else if (a.head_dim <= 96) GQ_AP(96);
    else GQ_AP(128);
#undef GQ_AP
    GQ_LAUNCH_CHECK();
    return GQ_OK;
}

}  // namespace

extern "C" int gq_attention_prompt(const gq_attention_prompt_args *args, gq_stream_t stream)
{
    GQ_REQUIRE(args, "gq_attention_prompt: NULL pointer");
    const gq_rows out = args->out, q = args->q, k = args->k, v = args->v;
    const int64_t dtype = args->dtype, n_tokens = args->n_tokens, n_heads = args->n_heads, n_kv_heads = args->n_kv_heads, head_dim = args->head_dim;
    const int64_t batch = args->batch;
    const int32_t *cu_seqlens = args->cu_seqlens;
    const float softmax_scale = (float)args->softmax_scale;
    GQ_REQUIRE(dtype == GQ_F16 || dtype == GQ_BF16, "gq_attention_prompt: dtype %lld is neither fp16 (0) nor bf16 (1)", (long long)dtype);
    GQ_REQUIRE(head_dim >= 8 && head_dim <= 128 && head_dim % 8 == 0, "gq_attention_prompt: head_dim %lld is not a multiple of 8 up to 128", (long long)head_dim);
    GQ_REQUIRE(n_heads > 0 && n_kv_heads > 0 && n_heads % n_kv_heads == 0 && n_heads <= 65536, "gq_attention_prompt: %lld query heads on %lld",
               (long long)n_heads, (long long)n_kv_heads);
    GQ_REQUIRE(n_tokens >= 0 && n_tokens < ((int64_t)1 << 30) && batch >= 0 && batch < (1 << 24), "gq_attention_prompt: bad number of tokens or sequences");
    GQ_REQUIRE(cu_seqlens || batch == 1 || n_tokens == 0, "gq_attention_prompt: %lld sequences need cu_seqlens", (long long)batch);
    GQ_REQUIRE(softmax_scale > 0.f && softmax_scale * AP_LOG2E < INFINITY, "gq_attention_prompt: the softmax scale must be positive and finite");
    if (n_tokens == 0 || batch == 0) return GQ_OK;
    GQ_REQUIRE(out.data && q.data && k.data && v.data, "gq_attention_prompt: NULL pointer");
    GQ_REQUIRE(out.token_stride % 8 == 0 && out.head_stride % 8 == 0 && q.token_stride % 8 == 0 && q.head_stride % 8 == 0 && k.token_stride % 8 == 0 &&
                   k.head_stride % 8 == 0 && v.token_stride % 8 == 0 && v.head_stride % 8 == 0,
               "gq_attention_prompt: strides must be multiples of 8 elements");
    GQ_REQUIRE(gq_rows_apart(out, n_tokens, n_heads, head_dim), "gq_attention_prompt: rows of out overlap");
    // a tile of 64 rows is addressed by 32-bit offsets, and a row must lie behind the one before it
    GQ_REQUIRE(n_tokens == 1 || (k.token_stride >= head_dim && v.token_stride >= head_dim && k.token_stride <= (1 << 23) && v.token_stride <= (1 << 23)),
               "gq_attention_prompt: token strides of k and v must be in head_dim..2^23");
    GQ_REQUIRE((((uintptr_t)out.data | (uintptr_t)q.data | (uintptr_t)k.data | (uintptr_t)v.data) & 15) == 0, "gq_attention_prompt: pointers must be 16-byte aligned");
    const int64_t n_items = cu_seqlens ? n_tokens / AP_Q + batch : gq_cdiv(n_tokens, AP_Q);
    GQ_REQUIRE(n_items * n_heads < GQ_MAX_THREADS / 256, "gq_attention_prompt: too many tokens for one call");
    PromptArgs a;
    a.q = q.data, a.k = k.data, a.v = v.data, a.out = out.data;
    a.q_tok = q.token_stride, a.q_head = q.head_stride, a.k_tok = k.token_stride, a.k_head = k.head_stride;
    a.v_tok = v.token_stride, a.v_head = v.head_stride, a.o_tok = out.token_stride, a.o_head = out.head_stride;
    if (n_tokens == 1) a.k_tok = a.v_tok = head_dim;   // (any stride may stand there)
    a.cu = cu_seqlens, a.n_tokens = n_tokens, a.batch = (int)batch, a.n_heads = (int)n_heads, a.group = (int)(n_heads / n_kv_heads);
    a.head_dim = (int)head_dim, a.n_items = (int)n_items, a.causal = args->causal != 0, a.scale = softmax_scale * AP_LOG2E;
    return dtype == GQ_F16 ? launch_prompt<_Float16>(a, (hipStream_t)stream) : launch_prompt<__bf16>(a, (hipStream_t)stream);
}
