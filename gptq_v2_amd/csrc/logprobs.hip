// Log probabilities of given tokens from rows of logits, with the entropy and the most likely alternatives.
//
// In units of log 2, y = x log2 e - M for any reference M near the maximum, S = sum 2^y and T = sum y 2^y over a row:
//   log p(t) = (y_t - log2 S) ln 2,     entropy = (log2 S - T / S) ln 2.
// (x times the rounded log2 e minus M is one fused operation, and M the same in both places: no error of M counts.)
// One workgroup takes one row and reads it once.  Every thread sums over its own elements with a reference of its own, to
// begin with the maximum of the first elements that its wave sees; it moves (S' = S f, T' = (T + d S) f for d = M - M',
// f = 2^d) only when an element is 2^8 above it, so that nearly all batches of chunks pass without a rescaling (following
// the maximum itself, some lane of the wave moves in nearly every one).  The sums cost 8 vector instructions an element,
// against the 11 that HBM's rate leaves time for.
//
// The alternatives need no second pass over the row.  Every thread knows the largest of its own elements and its chunk.
// Of 64 groups of threads, the k-th largest of the groups' largest bounds the k-th largest of the row from below, and only
// threads whose own largest is not below the bound (a dozen of 256) can hold larger ones: their elements are read again,
// by the whole workgroup, and the few at or above the bound ranked by counting.  Elements are compared by (value, -index)
// in one 64-bit word, so ties go to the lowest index; a thread's largest counts with the last index of its chunk, which
// can only lower the bound.
//
// Bound by HBM: rows * vocab elements in, a few words out; next to the vector instructions (86 % of the busy CUs' time).  4096 x
// 50272 bf16 with ten alternatives 89 us (4.6 TB/s; a read alone reaches 6), one row of 32000 fp16 with five 7.6 us (a launch and
// four dependent steps), on operands that no cache holds.
#include <type_traits>

#include "gq_common.h"

namespace {

constexpr int LP_MAX_TOP = 32;
constexpr int LP_GROUPS = 64;   // at least LP_MAX_TOP; one wave ranks them
constexpr int LP_LIST = 1024;   // candidates a workgroup ranks; a row with more takes the exhaustive path
constexpr float LP_LOG2E = 1.44269504088896340736f, LP_LN2 = 0.69314718055994530942f;

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

// Sums with their reference.  Elements of -inf add nothing.
struct Stat {
    float m, s, t;
    __device__ __forceinline__ void move(float to)
    {
        const float d = m - to, f = __builtin_amdgcn_exp2f(d);
        t = f == 0.f ? 0.f : fmaf(d, s, t) * f;   // (d s may overflow where f is 0)
        s *= f;
        m = to;
    }
    __device__ __forceinline__ void add(float x)
    {
        const float y = fmaf(x, LP_LOG2E, -m);
        const float e = __builtin_amdgcn_exp2f(y);
        s += e;
        t = fmaf(fmaxf(y, -160.f), e, t);   // (e is 0 there, y may be -inf)
    }
};

// The reference that belongs to an element; beyond 2e38 (a row of the type's lowest value) it is no longer near it, and
// such a row comes out as one without a sum, which is taken again
__device__ __forceinline__ float lp_reference(float x) { return fminf(fmaxf(x * LP_LOG2E, -3.0e38f), 3.0e38f); }

template <int WIDTH>
__device__ __forceinline__ float lp_max(float x)
{
#pragma unroll
    for (int off = WIDTH / 2; off > 0; off >>= 1) x = fmaxf(x, __shfl_xor(x, off, 64));
    return x;
}

template <int WIDTH>
__device__ __forceinline__ float lp_sum(float x)
{
#pragma unroll
    for (int off = WIDTH / 2; off > 0; off >>= 1) x += __shfl_xor(x, off, 64);
    return x;
}

template <typename T, int NT>
__global__ __launch_bounds__(NT) void token_logprobs_kernel(const T *__restrict__ logits, int64_t row_stride, int vocab,
                                                            const int64_t *__restrict__ tokens, int64_t ignore_index,
                                                            float *__restrict__ logprob, float *__restrict__ entropy, int top,
                                                            float *__restrict__ top_logprob, int64_t *__restrict__ top_token)
{
    constexpr int VEC = Chunk<T>::N;
    constexpr int UNROLL = 2;
    constexpr int WAVES = NT / 64;
    constexpr int PER_GROUP = NT / LP_GROUPS;
    __shared__ float sm_m[WAVES], sm_s[WAVES], sm_t[WAVES];
    __shared__ uint64_t sm_best[NT];
    __shared__ uint64_t sm_list[LP_LIST];
    __shared__ uint64_t sm_bound;
    __shared__ int sm_thread[NT];
    __shared__ int sm_threads, sm_count;

    const int64_t row = blockIdx.x;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const T *x = logits + row * row_stride;
    // elements before the first 16-byte boundary, whole chunks, elements behind the last
    int head = (int)(((16 - ((uintptr_t)x & 15)) & 15) / sizeof(T));
    head = head < vocab ? head : vocab;
    const int n_chunks = (vocab - head) / VEC;
    const int tail0 = head + n_chunks * VEC;
    const T *xc = x + head;

    int64_t token = 0;
    float x_token = 0.f;
    if (tid == 0) {
        token = tokens[row];
        if (token >= 0 && token < vocab) x_token = static_cast<float>(x[token]);
    }

    Stat st = {-3.0e38f, 0.f, 0.f};
    float best = -INFINITY;   // of this thread's chunks, and the chunk it is in
    int best_at = -1;
    const auto take = [&](int c, auto whole) {
        float f[UNROLL][VEC];
#pragma unroll
        for (int u = 0; u < UNROLL; ++u) {
            if (whole || c + u * NT < n_chunks) {
                load_chunk(xc + (c + u * NT) * VEC, f[u]);
            } else {
#pragma unroll
                for (int i = 0; i < VEC; ++i) f[u][i] = -INFINITY;
            }
        }
        float most = -INFINITY;   // (a maximum passes over NaN)
#pragma unroll
        for (int u = 0; u < UNROLL; ++u) {
            float of_chunk = -INFINITY;
#pragma unroll
            for (int i = 0; i < VEC; ++i) of_chunk = fmaxf(of_chunk, f[u][i]);
            if ((whole || c + u * NT < n_chunks) && (of_chunk > best || best_at < 0)) {
                best = of_chunk;
                best_at = c + u * NT;
            }
            most = fmaxf(most, of_chunk);
        }
        if (c < NT) st.m = lp_reference(lp_max<64>(most));   // the first batch
        const float m = lp_reference(most);
        if (__any(m > st.m + 8.f)) st.move(fmaxf(m, st.m));
#pragma unroll
        for (int u = 0; u < UNROLL; ++u)
#pragma unroll
            for (int i = 0; i < VEC; ++i) st.add(f[u][i]);
    };
    int c0 = 0;
    for (; c0 + UNROLL * NT <= n_chunks; c0 += UNROLL * NT) take(c0 + tid, std::true_type());
    if (c0 < n_chunks) take(c0 + tid, std::false_type());
    // the elements before the first and behind the last chunk
    if (tid < head + (vocab - tail0)) {
        const float v = static_cast<float>(x[tid < head ? tid : tail0 + tid - head]);
        const float m = lp_reference(v);
        if (m > st.m + 8.f) st.move(m);
        st.add(v);
    }

    const float top_m = lp_max<64>(st.m);
    if (lane == 0) sm_m[wave] = top_m;
    const uint64_t own = best_at >= 0 ? lp_key(best, head + best_at * VEC + VEC - 1) : 0;
    if (top > 0) {
        uint64_t key = own;
#pragma unroll
        for (int off = PER_GROUP / 2; off > 0; off >>= 1) {
            const uint64_t o = __shfl_xor((unsigned long long)key, off, 64);
            key = o > key ? o : key;
        }
        if (tid % PER_GROUP == 0) sm_best[tid / PER_GROUP] = key;
        if (tid == 0) {
            sm_count = sm_threads = 0;
            sm_bound = 0;
        }
    }
    __syncthreads();
    st.move(lp_max<WAVES>(sm_m[lane % WAVES]));
    st.s = lp_sum<64>(st.s);
    st.t = lp_sum<64>(st.t);
    if (lane == 0) {
        sm_s[wave] = st.s;
        sm_t[wave] = st.t;
    }
    // the top-th of the groups' largest (the words differ; of fewer groups with an element the bound stays 0)
    if (top > 0 && tid < LP_GROUPS) {
        const uint64_t mine = sm_best[tid];
        int rank = 0;
#pragma unroll 16
        for (int i = 0; i < LP_GROUPS; ++i) rank += sm_best[i] > mine;
        if (rank == top - 1) sm_bound = mine;
    }
    __syncthreads();
    st.s = lp_sum<WAVES>(sm_s[lane % WAVES]);
    st.t = lp_sum<WAVES>(sm_t[lane % WAVES]);
    // No sum: a row of numbers so large that their reference's own rounding (2^-24 of it) over- or underflows 2^y, of -inf
    // alone, with NaN or +inf.  It is taken again, from its maximum; the last three come out as NaN.
    float log_s = log2f(st.s), unit = LP_LN2, m = st.m;
    const bool odd = !(st.s > 0.f && st.s < INFINITY && fabsf(st.t) < INFINITY);
    if (odd) {
        __syncthreads();
        float most = -INFINITY;
        for (int i = tid; i < vocab; i += NT) most = fmaxf(most, static_cast<float>(x[i]));
        most = lp_max<64>(most);
        if (lane == 0) sm_m[wave] = most;
        __syncthreads();
        m = lp_max<WAVES>(sm_m[lane % WAVES]);
        float s = 0.f, t = 0.f;
        for (int i = tid; i < vocab; i += NT) {
            const float d = static_cast<float>(x[i]) - m, e = __builtin_amdgcn_exp2f(d * LP_LOG2E);
            s += e;
            t = fmaf(fmaxf(d, -3.0e38f), e, t);
        }
        s = lp_sum<64>(s);
        t = lp_sum<64>(t);
        if (lane == 0) {
            sm_s[wave] = s;
            sm_t[wave] = t;
        }
        __syncthreads();
        st.s = lp_sum<WAVES>(sm_s[lane % WAVES]);
        st.t = lp_sum<WAVES>(sm_t[lane % WAVES]);
        log_s = st.s > 0.f ? logf(st.s) : NAN;
        unit = 1.f;
    }
    const auto log_p = [&](float v) {
        const float y = odd ? v - m : fmaf(v, LP_LOG2E, -m);
        // (a number near the type's lowest is out of range in units of log 2)
        return y == -INFINITY ? v - (m + log_s) * unit : (y - log_s) * unit;
    };
    if (tid == 0) {
        float lp = NAN;
        if (token == ignore_index) lp = 0.f;
        else if (token >= 0 && token < vocab) lp = log_p(x_token);
        logprob[row] = lp;
        entropy[row] = (log_s - st.t / st.s) * unit;
    }
    if (top == 0) return;
    const uint64_t bound = sm_bound;
    const float bound_value = lp_value(bound);   // (a bound of 0 is NaN: below nothing)
    const auto offer = [&](float v, int index) {
        if (v < bound_value) return;
        const uint64_t key = lp_key(v, index);
        if (key >= bound) {
            const int at = atomicAdd(&sm_count, 1);
            if (at < LP_LIST) sm_list[at] = key;
        }
    };
    if (own != 0 && own >= bound) sm_thread[atomicAdd(&sm_threads, 1)] = tid;
    __syncthreads();
    const int per_thread = (n_chunks + NT - 1) / NT, n_again = sm_threads * per_thread;
    for (int i = tid; i < n_again; i += NT) {
        const int s = i / per_thread, ch = sm_thread[s] + (i - s * per_thread) * NT;
        if (ch >= n_chunks) continue;
        float g[VEC], most = -INFINITY;
        load_chunk(xc + ch * VEC, g);
#pragma unroll
        for (int j = 0; j < VEC; ++j) most = fmaxf(most, g[j]);
        if (most < bound_value) continue;
#pragma unroll
        for (int j = 0; j < VEC; ++j) offer(g[j], head + ch * VEC + j);
    }
    if (tid < head + (vocab - tail0)) {
        const int idx = tid < head ? tid : tail0 + tid - head;
        offer(static_cast<float>(x[idx]), idx);
    }
    __syncthreads();
    const int count = sm_count;
    if (count <= LP_LIST && !odd) {
        for (int i = tid; i < count; i += NT) {
            const uint64_t key = sm_list[i];
            int r = 0;
            for (int j = 0; j < count; ++j) r += sm_list[j] > key;
            if (r < top) {
                top_logprob[row * top + r] = log_p(lp_value(key));
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
            top_logprob[row * top + r] = log_p(lp_value(last));
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
    // 16 waves a row up to 512 rows that have a chunk or two for each thread (two such workgroups a CU at once), else 4.  16
    // and 4 waves on operands that no cache holds, in us: 50272 words of bf16 with ten alternatives 10.9 and 16.6 for 64 rows,
    // 12.1 and 17.8 for 256, 16.1 and 18.9 for 300, 18.0 and 20.8 for 512, 25.2 and 24.2 for 640, 32.2 and 30.9 for 1024; 17000
    // words 12.2 and 11.7 for 512 rows, 21.6 and 14.7 for 1024.  Only rows of 200 KB and more would have 16 waves beyond (128256
    // words of fp32, 1024 rows: 97 and 127).
    if (n_rows <= 512 && vocab * (int64_t)sizeof(T) >= 32768) GQ_LP(1024);
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
    GQ_REQUIRE(n_rows >= 0 && n_rows < GQ_MAX_THREADS / 256, "gq_token_logprobs: bad row count %lld", (long long)n_rows);
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
