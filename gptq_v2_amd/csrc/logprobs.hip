// Log probabilities of given tokens from rows of logits, with the entropy and the most likely alternatives.
//
// With m = max x, S = sum e^(x - m) and T = sum (x - m) e^(x - m) over a row:
//   log p(t) = (x_t - m) - log S,     entropy = log S - T / S.
// One workgroup takes one row and reads it once: every thread keeps a running (m, S, T) of its own elements and
// rescales it when m grows (S' = S f, T' = (T + d S) f for d = m - m', f = e^d), the workgroup joins them.
//
// The alternatives need no second pass over the row.  The threads form 64 groups, a group's elements a stripe of the
// row, and the running maxima give each stripe's best element.  The k-th largest of the 64 bounds the k-th largest of
// the row from below, and only the k stripes at or above that bound can hold larger elements: those (k / 64 of the row,
// from the cache) are read again and the few elements at or above the bound ranked by counting.  Elements are compared
// by (value, -index) in one 64-bit word, so ties go to the lowest index.
//
// Bound by HBM: rows * vocab elements in, a few words out.
#include "gq_common.h"

namespace {

constexpr int LP_MAX_TOP = 32;
constexpr int LP_GROUPS = 64;   // at least LP_MAX_TOP; one wave ranks them
constexpr int LP_LIST = 1024;   // candidates a workgroup ranks; a row with more takes the exhaustive path
constexpr float LP_LOG2E = 1.44269504088896340736f;

template <typename T> struct Chunk { static constexpr int N = 16 / sizeof(T); };

template <typename T>
__device__ __forceinline__ void load_chunk(const T *p, float (&x)[Chunk<T>::N])
{
    const u32x4 raw = *reinterpret_cast<const u32x4 *>(p);
    T v[Chunk<T>::N];
    __builtin_memcpy(v, &raw, 16);
#pragma unroll
    for (int i = 0; i < Chunk<T>::N; ++i) x[i] = static_cast<float>(v[i]);
}

// (value, -index) as one word that compares as an integer: NaN above +inf (as a sort orders it), -0 equal to 0;
// below ~0 for every element
__device__ __forceinline__ uint64_t lp_key(float x, uint32_t index)
{
    uint32_t b = __float_as_uint(x);
    if (x == 0.f) b = 0;
    b = (b & 0x80000000u) ? ~b : (b | 0x80000000u);
    if (x != x) b = 0xffffffffu;
    return ((uint64_t)b << 32) | (0xfffffffeu - index);
}

__device__ __forceinline__ float lp_value(uint64_t key)
{
    const uint32_t b = (uint32_t)(key >> 32);
    return __uint_as_float((b & 0x80000000u) ? (b & 0x7fffffffu) : ~b);
}

struct Stat {
    float m, s, t;
};

// One more element range under a common maximum.  -inf is held apart: e^(-inf - m) is 0 and adds nothing, and a
// thread that has seen nothing else (m = -inf) must not turn that into NaN.
__device__ __forceinline__ Stat lp_join(Stat a, Stat b)
{
    const float m = fmaxf(a.m, b.m);
    if (m == -INFINITY) return {m, a.s + b.s, 0.f};   // the sums are 0, or NaN from a NaN element
    const float da = a.m - m, db = b.m - m;
    const float fa = __builtin_amdgcn_exp2f(da * LP_LOG2E), fb = __builtin_amdgcn_exp2f(db * LP_LOG2E);
    const float ta = a.m == -INFINITY ? 0.f : fmaf(da, a.s, a.t) * fa;
    const float tb = b.m == -INFINITY ? 0.f : fmaf(db, b.s, b.t) * fb;
    return {m, a.s * fa + b.s * fb, ta + tb};
}

__device__ __forceinline__ Stat lp_shuffle(Stat a, int off)
{
    return {__shfl_xor(a.m, off, 64), __shfl_xor(a.s, off, 64), __shfl_xor(a.t, off, 64)};
}

template <int N>
__device__ __forceinline__ void lp_take(const float (&x)[N], uint32_t index, Stat &st, uint32_t &best)
{
    float cm = -INFINITY;
#pragma unroll
    for (int i = 0; i < N; ++i)
        cm = fmaxf(cm, x[i]);
    if (cm > st.m || best == 0xffffffffu) {
        int at = 0;
#pragma unroll
        for (int i = N - 1; i >= 0; --i)
            if (x[i] == cm) at = i;
        best = index + at;
        if (st.m != -INFINITY) {
            const float d = st.m - cm, f = __builtin_amdgcn_exp2f(d * LP_LOG2E);
            st.t = fmaf(d, st.s, st.t) * f;
            st.s *= f;
        }
        st.m = cm;
    }
    const float ref = st.m == -INFINITY ? 0.f : st.m;
#pragma unroll
    for (int i = 0; i < N; ++i) {
        const float d = x[i] - ref;
        const float e = __builtin_amdgcn_exp2f(d * LP_LOG2E);
        st.s += e;
        st.t = fmaf(fmaxf(d, -3.0e38f), e, st.t);   // -inf * 0 counts as 0
    }
}

template <typename T, int NT>
__global__ __launch_bounds__(NT) void token_logprobs_kernel(const T *__restrict__ logits, int64_t row_stride, int vocab,
                                                            const int64_t *__restrict__ tokens, int64_t ignore_index,
                                                            float *__restrict__ logprob, float *__restrict__ entropy, int top,
                                                            float *__restrict__ top_logprob, int64_t *__restrict__ top_token)
{
    constexpr int VEC = Chunk<T>::N;
    constexpr int UNROLL = 4;
    constexpr int WAVES = NT / 64;
    constexpr int PER_GROUP = NT / LP_GROUPS;
    __shared__ float sm_m[WAVES], sm_s[WAVES], sm_t[WAVES];
    __shared__ uint64_t sm_best[NT];
    __shared__ uint64_t sm_list[LP_LIST];
    __shared__ uint64_t sm_bound;
    __shared__ int sm_stripe[LP_MAX_TOP];
    __shared__ int sm_count;

    const int64_t row = blockIdx.x;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const T *x = logits + row * row_stride;
    // elements before the first 16-byte boundary, whole chunks, elements behind the last
    int head = (int)(((16 - ((uintptr_t)x & 15)) & 15) / sizeof(T));
    head = head < vocab ? head : vocab;
    const int n_chunks = (vocab - head) / VEC;
    const int tail0 = head + n_chunks * VEC;
    const T *xc = x + head;

    Stat st = {-INFINITY, 0.f, 0.f};
    uint32_t best = 0xffffffffu;
    if (tid < head) {
        const float one[1] = {static_cast<float>(x[tid])};
        lp_take<1>(one, tid, st, best);
    }
    int c = tid;
    for (; c + (UNROLL - 1) * NT < n_chunks; c += UNROLL * NT) {
        float f[UNROLL][VEC];
#pragma unroll
        for (int u = 0; u < UNROLL; ++u) load_chunk(xc + (int64_t)(c + u * NT) * VEC, f[u]);
#pragma unroll
        for (int u = 0; u < UNROLL; ++u) lp_take<VEC>(f[u], head + (c + u * NT) * VEC, st, best);
    }
    for (; c < n_chunks; c += NT) {
        float f[VEC];
        load_chunk(xc + (int64_t)c * VEC, f);
        lp_take<VEC>(f, head + c * VEC, st, best);
    }
    if (tid < vocab - tail0) {
        const float one[1] = {static_cast<float>(x[tail0 + tid])};
        lp_take<1>(one, tail0 + tid, st, best);
    }

    if (top > 0) {
        uint64_t key = best == 0xffffffffu ? 0 : lp_key(st.m, best);
#pragma unroll
        for (int off = PER_GROUP / 2; off > 0; off >>= 1) {
            const uint64_t o = __shfl_xor((unsigned long long)key, off, 64);
            key = o > key ? o : key;
        }
        if (tid % PER_GROUP == 0) sm_best[tid / PER_GROUP] = key;
        if (tid == 0) sm_count = 0;
    }
#pragma unroll
    for (int off = 32; off > 0; off >>= 1) st = lp_join(st, lp_shuffle(st, off));
    if (lane == 0) {
        sm_m[wave] = st.m;
        sm_s[wave] = st.s;
        sm_t[wave] = st.t;
    }
    __syncthreads();
    st = {sm_m[0], sm_s[0], sm_t[0]};
    for (int w = 1; w < WAVES; ++w) st = lp_join(st, {sm_m[w], sm_s[w], sm_t[w]});
    // no element, only -inf, a NaN or +inf: not a distribution
    const bool bad = !(st.m > -INFINITY) || !(st.s > 0.f);
    const float log_s = bad ? NAN : logf(st.s);
    if (tid == 0) {
        const int64_t t = tokens[row];
        float lp = NAN;
        if (t == ignore_index) lp = 0.f;
        else if (t >= 0 && t < vocab) lp = (static_cast<float>(x[t]) - st.m) - log_s;
        logprob[row] = lp;
        entropy[row] = log_s - st.t / st.s;
    }
    if (top == 0) return;

    // ranks of the groups' best (the words differ, but for the zeros of groups without an element)
    if (tid < LP_GROUPS) {
        const uint64_t mine = sm_best[tid];
        int rank = 0;
        for (int i = 0; i < LP_GROUPS; ++i) {
            const uint64_t o = sm_best[i];
            rank += (o > mine) || (o == mine && i < tid);
        }
        if (rank < top) sm_stripe[rank] = tid;
        if (rank == top - 1) sm_bound = mine;
    }
    __syncthreads();
    const uint64_t bound = sm_bound;
    const int per_stripe = (n_chunks + NT - 1) / NT * PER_GROUP;
    for (int i = tid; i < top * per_stripe; i += NT) {
        const int s = i / per_stripe, j = i - s * per_stripe;
        const int ch = sm_stripe[s] * PER_GROUP + (j % PER_GROUP) + (j / PER_GROUP) * NT;
        if (ch >= n_chunks) continue;
        float f[VEC];
        load_chunk(xc + (int64_t)ch * VEC, f);
#pragma unroll
        for (int j2 = 0; j2 < VEC; ++j2) {
            const uint64_t key = lp_key(f[j2], head + ch * VEC + j2);
            if (key >= bound) {
                const int at = atomicAdd(&sm_count, 1);
                if (at < LP_LIST) sm_list[at] = key;
            }
        }
    }
    if (tid < head + (vocab - tail0)) {
        const int idx = tid < head ? tid : tail0 + tid - head;
        const uint64_t key = lp_key(static_cast<float>(x[idx]), idx);
        if (key >= bound) {
            const int at = atomicAdd(&sm_count, 1);
            if (at < LP_LIST) sm_list[at] = key;
        }
    }
    __syncthreads();
    const int count = sm_count;
    if (count <= LP_LIST && !bad) {
        for (int i = tid; i < count; i += NT) {
            const uint64_t key = sm_list[i];
            int r = 0;
            for (int j = 0; j < count; ++j) r += sm_list[j] > key;
            if (r < top) {
                top_logprob[row * top + r] = (lp_value(key) - st.m) - log_s;
                top_token[row * top + r] = (int64_t)(0xfffffffeu - (uint32_t)key);
            }
        }
        return;
    }
    // More candidates than the list holds (the row's largest elements crowd into few stripes), or a row with NaN
    // (which a running maximum passes over): one search of the row for each alternative.
    uint64_t last = ~0ull;
    for (int r = 0; r < top; ++r) {
        uint64_t found = 0;
        for (int i = tid; i < vocab; i += NT) {
            const uint64_t key = lp_key(static_cast<float>(x[i]), i);
            if (key < last && key > found) found = key;
        }
        sm_best[tid] = found;
        __syncthreads();
        for (int half = NT / 2; half > 0; half >>= 1) {
            if (tid < half) sm_best[tid] = sm_best[tid] > sm_best[tid + half] ? sm_best[tid] : sm_best[tid + half];
            __syncthreads();
        }
        last = sm_best[0];
        __syncthreads();
        if (tid == 0) {
            top_logprob[row * top + r] = bad ? NAN : (lp_value(last) - st.m) - log_s;
            top_token[row * top + r] = (int64_t)(0xfffffffeu - (uint32_t)last);
        }
    }
}

template <typename T>
int launch_logprobs(const void *logits, int64_t n_rows, int64_t row_stride, int64_t vocab, const int64_t *tokens, int64_t ignore_index,
                    float *logprob, float *entropy, int top, float *top_logprob, int64_t *top_token, hipStream_t s)
{
#define GQ_LP(NT)                                                                                                                      \
    hipLaunchKernelGGL((token_logprobs_kernel<T, NT>), dim3((unsigned)n_rows), dim3(NT), 0, s, (const T *)logits, row_stride, (int)vocab, \
                       tokens, ignore_index, logprob, entropy, top, top_logprob, top_token)
    if (n_rows <= 512) GQ_LP(1024);
    else GQ_LP(256);
#undef GQ_LP
    GQ_LAUNCH_CHECK();
    return GQ_OK;
}

}  // namespace

extern "C" int gq_token_logprobs(const gq_token_logprobs_args *args, gq_stream_t stream)
{
    GQ_REQUIRE(args, "gq_token_logprobs: NULL pointer");
    const void *logits = args->logits;
    const int64_t dtype = args->dtype, n_rows = args->n_rows, row_stride = args->row_stride, vocab = args->vocab, ignore_index = args->ignore_index;
    const int64_t *tokens = args->tokens;
    float *logprob = args->logprob, *entropy = args->entropy, *top_logprob = args->top_logprob;
    int64_t *top_token = args->top_token;
    GQ_REQUIRE(dtype == GQ_F16 || dtype == GQ_BF16 || dtype == GQ_F32, "gq_token_logprobs: dtype %lld is none of fp16 (0), bf16 (1), fp32 (2)",
               (long long)dtype);
    GQ_REQUIRE(n_rows >= 0 && n_rows < ((int64_t)1 << 31), "gq_token_logprobs: bad row count %lld", (long long)n_rows);
    GQ_REQUIRE(vocab > 0 && vocab <= (1 << 30), "gq_token_logprobs: vocab must be in 1..2^30");
    GQ_REQUIRE(args->top >= 0 && args->top <= LP_MAX_TOP && args->top <= vocab, "gq_token_logprobs: %lld alternatives: 0..%d of the vocabulary can be asked for",
               (long long)args->top, LP_MAX_TOP);
    const int top = (int)args->top;
    GQ_REQUIRE(row_stride >= vocab || n_rows <= 1, "gq_token_logprobs: rows of %lld overlap at a stride of %lld", (long long)vocab, (long long)row_stride);
    if (n_rows == 0) return GQ_OK;
    GQ_REQUIRE(logits && tokens && logprob && entropy && (top == 0 || (top_logprob && top_token)), "gq_token_logprobs: NULL pointer");
    GQ_REQUIRE(((uintptr_t)logits & (dtype == GQ_F32 ? 3 : 1)) == 0, "gq_token_logprobs: logits are not aligned to their type");
    GQ_REQUIRE((((uintptr_t)tokens | (uintptr_t)top_token) & 7) == 0 && (((uintptr_t)logprob | (uintptr_t)entropy | (uintptr_t)top_logprob) & 3) == 0,
               "gq_token_logprobs: tokens or outputs are not aligned to their type");
    const hipStream_t s = (hipStream_t)stream;
    if (dtype == GQ_F16)
        return launch_logprobs<_Float16>(logits, n_rows, row_stride, vocab, tokens, ignore_index, logprob, entropy, top, top_logprob, top_token, s);
    if (dtype == GQ_BF16)
        return launch_logprobs<__bf16>(logits, n_rows, row_stride, vocab, tokens, ignore_index, logprob, entropy, top, top_logprob, top_token, s);
    return launch_logprobs<float>(logits, n_rows, row_stride, vocab, tokens, ignore_index, logprob, entropy, top, top_logprob, top_token, s);
}
