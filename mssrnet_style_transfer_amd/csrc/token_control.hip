// Control of the next token's logits: penalties for tokens of the history, a bias, a grammar's mask, no repeated n-grams;
// either the new logits or only the pick (the largest) leaves.
//
// Per row, in fp32 with every step rounded:
//   v in the history:  x = x > 0 ? x / repetition : x * repetition
//   its count, over the history from prompt_lengths on, above 0:  x = x - (frequency * count + presence)
//   x = x + bias[v];   x = -inf where the mask's bit is 0 or v would complete an n-gram of the history
// Bound by memory: the logits once, written once or not at all.  A block owns a chunk of a row: it walks the history
// first and marks the chunk's words in LDS (count, seen, banned; 16 bits a word while counts fit, so that a chunk can be
// 32768 words: every chunk of a row walks the whole history), then streams the logits, 8 words a thread.
// Measured: 128 rows x 50001 fp32 words, history 300, new logits (52 MB) 15.4 us, 3.4 TB/s; 64 x 131071 bf16, history 2000 with
// 4-grams (35 MB) 13.9 us; the pick of 512 x 9606 bf16 (10 MB) 8.7 us and of one row 5.5 us, where latency counts: a launch 2.5,
// the logits 1.4, the history's walk (clear, walk, two barriers) 1.1 (1.8 with two blocks a CU).
#include "common.hpp"
#include "kv4.hpp"      // IdxTable

namespace mssr {

constexpr int TC_THREADS = 1024;
constexpr int TC_UNIT = TC_THREADS * 8;          // a chunk is a multiple of this
constexpr int TC_LDS = 65536;                    // bytes of marks
constexpr int64_t TC_MAX_GRID = (1 << 22) - 1;   // blocks of 1024 threads: a grid has fewer than 2^32 threads
constexpr int64_t TC_MAX_T = 0x3fffffff;
constexpr int64_t TC_MAX_LD = (int64_t)1 << 36;  // of rows: 2^22 of them stay within 64-bit offsets

// a word's mark: the two top bits of M (16 or 32 bits) are flags, the rest counts
template <typename M> struct Mark {
    static constexpr int bits = 8 * sizeof(M), per = 4 / sizeof(M);
    static constexpr uint32_t seen = 1u << (bits - 1), banned = 1u << (bits - 2), count = banned - 1;
    static __device__ __forceinline__ int shift(int i) { return sizeof(M) == 2 ? 16 * (i & 1) : 0; }
};
constexpr int64_t TC_MARK16_T = Mark<uint16_t>::count;      // the longest history whose counts fit

struct TokenControlArgs {
    const void* logits;
    void* out;                                   // new logits, or null
    int64_t ld, ldo, V;
    int B, chunk, chunks;
    const void* history;
    int64_t h_bs, h_ts;
    int h64;
    int64_t T;
    IdxTable lengths, prompt;
    const float *repetition, *frequency, *presence;      // per row, or null
    float repetition0, frequency0, presence0;
    int ngram;
    const float* bias;
    int64_t bias_bs;
    const uint32_t* allowed;
    int64_t states, words;
    IdxTable state;
    int state_mode;                              // 0: row 0, 1: row b, 2: state[b]
    void* ids;                                   // the pick, or null
    int ids64;
    int64_t empty;
    unsigned long long* part;                    // [B][chunks] packed picks
};

__device__ __forceinline__ int64_t tc_token(const TokenControlArgs& a, int64_t b, int64_t t) {
    const int64_t at = b * a.h_bs + t * a.h_ts;
    return a.h64 ? ((const int64_t*)a.history)[at] : (int64_t)((const int32_t*)a.history)[at];
}

// larger float -> larger key; -0 equals +0, NaN is above everything (as in torch.argmax); ties go to the lower index
__device__ __forceinline__ unsigned long long tc_key(float x, uint32_t v) {
    const uint32_t u = __builtin_bit_cast(uint32_t, x + 0.0f);
    const uint32_t o = x != x ? 0xffffffffu : ((u & 0x80000000u) ? ~u : (u | 0x80000000u));
    return ((unsigned long long)o << 32) | (uint32_t)~v;
}
constexpr uint32_t TC_NEG_INF_KEY = ~0xff800000u;

__device__ __forceinline__ unsigned long long tc_wave_max(unsigned long long k) {
#pragma unroll
    for (int d = 32; d; d >>= 1) {
        const unsigned long long o = __shfl_xor(k, d);
        k = o > k ? o : k;
    }
    return k;
}
__device__ __forceinline__ void tc_store_pick(const TokenControlArgs& a, int64_t b, unsigned long long k) {
    const int64_t id = (uint32_t)(k >> 32) <= TC_NEG_INF_KEY ? a.empty : (int64_t)(uint32_t)~(uint32_t)k;
    if (a.ids64) ((int64_t*)a.ids)[b] = id;
    else ((int32_t*)a.ids)[b] = (int32_t)id;
}

// 8 words of a row on their way: logits as they lie (rows start anywhere: the vocabulary's size may be odd), bias, mask bits
template <typename T>
struct Words {
    typedef T raw_t __attribute__((ext_vector_type(8)));
    raw_t x;
    float add[8];
    uint8_t open;
    __device__ __forceinline__ void load(const T* row, const float* bias, int i, int n) {
        if (i >= n) return;
        if (i + 8 <= n) {
            __builtin_memcpy(&x, row + i, sizeof(x));
            if (bias) __builtin_memcpy(add, bias + i, 32);
        } else {
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                x[e] = i + e < n ? row[i + e] : (T)0.f;
                add[e] = bias && i + e < n ? bias[i + e] : 0.f;
            }
        }
    }
    __device__ __forceinline__ void load_mask(const uint8_t* mask, int i, int n) {
        open = mask && i < n ? mask[i >> 3] : (uint8_t)0xff;
    }
};

template <typename T, typename M>
__global__ __launch_bounds__(TC_THREADS, sizeof(M) == 2 ? 8 : 4) void token_control_kernel(TokenControlArgs a) {
#pragma clang fp contract(off)
    extern __shared__ __align__(16) uint32_t mark[];
    __shared__ unsigned long long best[TC_THREADS / 64];
    const uint32_t b = blockIdx.x / (uint32_t)a.chunks;
    const int ci = (int)(blockIdx.x - b * (uint32_t)a.chunks), tid = threadIdx.x;
    const int64_t v0 = (int64_t)ci * a.chunk;
    const int n = (int)(a.V - v0 < a.chunk ? a.V - v0 : a.chunk);
    const T* x = (const T*)a.logits + b * a.ld + v0;
    const float* bias = a.bias ? a.bias + b * a.bias_bs + v0 : nullptr;
    T* out = a.out ? (T*)a.out + b * a.ldo + v0 : nullptr;
    // Everything whose address is known now is requested now, logits first: the row's words wait under the history's walk,
    // the history's first tokens under the clearing of the marks.
    Words<T> w[2];
    w[0].load(x, bias, 8 * tid, n);
    w[1].load(x, bias, 8 * tid + TC_UNIT, n);
    int64_t tok = -1, before = 0, last = 0, len = 0, from = 0;
    const bool grams = a.ngram > 1;
    if (a.history) {
        if (tid < a.T) {
            tok = tc_token(a, b, tid);
            if (grams && tid > 0) before = tc_token(a, b, tid - 1);
        }
        len = a.lengths.p ? a.lengths.at(b) : a.T;
        len = len < 0 ? 0 : (len > a.T ? a.T : len);
        from = a.prompt.at(b);
        if (grams && len > 0) last = tc_token(a, b, len - 1);
    }
    const uint8_t* mask = nullptr;
    bool closed = false;
    if (a.allowed) {
        const int64_t st = a.state_mode == 0 ? 0 : a.state_mode == 1 ? b : a.state.at(b);
        if (st >= a.states) closed = true;       // not a state of the table: nothing is allowed
        else if (st >= 0) mask = reinterpret_cast<const uint8_t*>(a.allowed + st * a.words) + (v0 >> 3);
    }
    w[0].load_mask(mask, 8 * tid, n);
    w[1].load_mask(mask, 8 * tid + TC_UNIT, n);
    const float rep = a.repetition ? a.repetition[b] : a.repetition0;
    const float freq = a.frequency ? a.frequency[b] : a.frequency0;
    const float pres = a.presence ? a.presence[b] : a.presence0;

    if (a.history) {
        for (int i = tid; i < (n + 4 * Mark<M>::per - 1) / (4 * Mark<M>::per); i += TC_THREADS)
            reinterpret_cast<u32x4*>(mark)[i] = u32x4{0, 0, 0, 0};
        __syncthreads();
        for (int64_t t = tid; t < len; t += TC_THREADS) {
            if (t != tid) {
                tok = tc_token(a, b, t);
                if (grams) before = tc_token(a, b, t - 1);
            }
            const int64_t at = tok - v0;
            if (at < 0 || at >= n) continue;
            const int i = (int)at, sh = Mark<M>::shift(i);
            uint32_t* word = &mark[i / Mark<M>::per];
            if (t >= from) atomicAdd(word, 1u << sh);
            uint32_t flags = Mark<M>::seen;
            if (a.ngram == 1) flags |= Mark<M>::banned;
            if (grams && t >= a.ngram - 1 && before == last) {
                bool same = true;
                for (int j = 2; j < a.ngram && same; ++j) same = tc_token(a, b, t - j) == tc_token(a, b, len - j);
                if (same) flags |= Mark<M>::banned;
            }
            atomicOr(word, flags << sh);
        }
        __syncthreads();
    }
    float most = -INFINITY;                      // this thread's largest word, NaN if it met one (the first stays)
    uint32_t at = 0;
    auto words = [&](const Words<T>& q, int i) {
        if (i >= n) return;
        uint32_t ban = closed ? 0xffu : (uint32_t)(uint8_t)~q.open;
        float y[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) y[e] = to_f(q.x[e]);
        if (a.history) {
            uint32_t m[8 / Mark<M>::per], any = 0;
            __builtin_memcpy(m, __builtin_assume_aligned(&mark[i / Mark<M>::per], 16), sizeof(m));
#pragma unroll
            for (int e = 0; e < 8 / Mark<M>::per; ++e) any |= m[e];
            if (any) {                           // rare: few words of the vocabulary are in a history
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    const uint32_t mk = (m[e / Mark<M>::per] >> Mark<M>::shift(e)) & (Mark<M>::seen | (Mark<M>::seen - 1));
                    if (!mk) continue;
                    const uint32_t c = mk & Mark<M>::count;
                    const float z = y[e] > 0.f ? y[e] / rep : y[e] * rep;
                    y[e] = c ? z - (freq * (float)c + pres) : z;     // (an infinite rate leaves the words that it does not count)
                    if (mk & Mark<M>::banned) ban |= 1u << e;
                }
            }
        }
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            if (bias) y[e] = y[e] + q.add[e];
            const float z = y[e];
            y[e] = (ban >> e) & 1u ? -INFINITY : z;
        }
        if (out) {
            if (i + 8 <= n) {
                typename Words<T>::raw_t r;
#pragma unroll
                for (int e = 0; e < 8; ++e) r[e] = from_f<T>(y[e]);
                __builtin_memcpy(out + i, &r, sizeof(r));
            } else {
                for (int e = 0; e < 8; ++e)
                    if (i + e < n) out[i + e] = from_f<T>(y[e]);
            }
        }
        if (a.ids) {
#pragma unroll
            for (int e = 0; e < 8; ++e) {        // ascending: a tie keeps the lower index
                const bool take = !(y[e] <= most) && most == most && i + e < n;
                most = take ? y[e] : most;
                at = take ? (uint32_t)(i + e) : at;
            }
        }
    };
    for (int i = 8 * tid; i < n; i += 2 * TC_UNIT) {
#pragma unroll
        for (int p = 0; p < 2; ++p) {
            const int j = i + p * TC_UNIT, next = j + 2 * TC_UNIT;
            words(w[p], j);
            w[p].load(x, bias, next, n);
            w[p].load_mask(mask, next, n);
        }
    }
    if (!a.ids) return;
    unsigned long long top = tc_key(most, (uint32_t)v0 + at);
    top = tc_wave_max(top);
    if ((tid & 63) == 0) best[tid >> 6] = top;
    __syncthreads();
    if (tid >= 64) return;
    top = tc_wave_max(tid < TC_THREADS / 64 ? best[tid] : 0);
    if (tid) return;
    if (a.chunks == 1) tc_store_pick(a, b, top);
    else a.part[blockIdx.x] = top;
}

__global__ __launch_bounds__(64) void token_pick_join_kernel(TokenControlArgs a) {
    unsigned long long top = 0;
    for (int i = threadIdx.x; i < a.chunks; i += 64) {
        const unsigned long long k = a.part[(int64_t)blockIdx.x * a.chunks + i];
        top = k > top ? k : top;
    }
    top = tc_wave_max(top);
    if (threadIdx.x == 0) tc_store_pick(a, blockIdx.x, top);
}

struct TcShape { int chunk, chunks; bool wide; };

// How rows are cut.  A chunk's marks are 64 KB at most.  Every chunk walks the row's history, so there are only as many as
// give 256 blocks, 512 where the walk is one round (64 rows x 131071 words, history 2000: 14.0 us with 256, 16.2 with 512;
// 128 x 50001, history 300: 17.6 and 15.1).  A pick of a row that fits a block's first loads is one chunk: joining takes
// another launch (9606 words: 5.4 us against 6.6).
static TcShape tc_shape(int64_t B, int64_t V, int64_t T, bool pick) {
    TcShape s;
    s.wide = T > TC_MARK16_T;
    const int64_t largest = TC_LDS / (s.wide ? 4 : 2), least = (V + largest - 1) / largest, most = (V + TC_UNIT - 1) / TC_UNIT;
    int64_t c = pick && V <= 2 * TC_UNIT ? 1 : ((T <= TC_THREADS ? 512 : 256) + B - 1) / B;
    c = c < least ? least : (c > most ? most : c);
    s.chunk = (int)(((V + c - 1) / c + TC_UNIT - 1) / TC_UNIT * TC_UNIT);
    s.chunks = (int)((V + s.chunk - 1) / s.chunk);
    return s;
}

// New logits take the old ones' place exactly, or share no element with them: apart as wholes, or other columns of equally
// strided rows.
static bool tc_apart(const mssr_token_control_desc* d) {
    const int64_t es = d->dtype == MSSR_F32 ? 4 : 2, x = (int64_t)(intptr_t)d->logits, y = (int64_t)(intptr_t)d->out;
    if (x == y) return d->B == 1 || d->ld == d->ldo;
    const int64_t row = d->V * es;
    if (x + (d->B - 1) * d->ld * es + row <= y || y + (d->B - 1) * d->ldo * es + row <= x) return true;
    if (d->ld != d->ldo) return false;
    const int64_t gap = ((y - x) % (d->ld * es) + d->ld * es) % (d->ld * es);
    return gap >= row && gap <= d->ld * es - row;
}

// The new logits and the bias have no byte in common: a block reads its bias while others write.
static bool tc_bias_apart(const mssr_token_control_desc* d) {
    const int64_t es = d->dtype == MSSR_F32 ? 4 : 2, y = (int64_t)(intptr_t)d->out, z = (int64_t)(intptr_t)d->bias;
    return y + ((d->B - 1) * d->ldo + d->V) * es <= z || z + ((d->B - 1) * d->bias_bs + d->V) * 4 <= y;
}

template <typename T>
static void tc_launch(const TokenControlArgs& a, bool wide, unsigned grid, unsigned lds, hipStream_t st) {
    if (wide) token_control_kernel<T, uint32_t><<<grid, TC_THREADS, lds, st>>>(a);
    else token_control_kernel<T, uint16_t><<<grid, TC_THREADS, lds, st>>>(a);
}

}  // namespace mssr

using namespace mssr;

extern "C" int64_t mssr_token_control_scratch(int64_t B, int64_t V, int64_t T) {
    if (B < 1 || V < 1 || V > INT32_MAX || T < 0 || T > TC_MAX_T) return -1;
    const TcShape s = tc_shape(B, V, T, true);
    return s.chunks > 1 ? B * s.chunks * (int64_t)sizeof(unsigned long long) : 0;
}

extern "C" int mssr_token_control(const mssr_token_control_desc* d, void* stream) {
    MSSR_REQUIRE(d, "token_control: no descriptor");
    MSSR_REQUIRE(d->B >= 0 && d->V >= 1 && d->V <= INT32_MAX && d->ld >= d->V && d->ld <= TC_MAX_LD, "token_control: logits [%lld, %lld], row stride %lld",
                 (long long)d->B, (long long)d->V, (long long)d->ld);
    MSSR_REQUIRE(valid_dtype(d->dtype), "token_control: dtype %d", d->dtype);
    if (d->B == 0) return MSSR_OK;
    MSSR_REQUIRE(d->logits && (d->out || d->ids), "token_control: null operand");
    MSSR_REQUIRE(!d->out || (d->ldo >= d->V && d->ldo <= TC_MAX_LD), "token_control: row stride %lld of the new logits", (long long)d->ldo);
    MSSR_REQUIRE(!d->ids || (d->index_bits & 16) || (d->empty >= INT32_MIN && d->empty <= INT32_MAX),
                 "token_control: %lld for an empty row does not fit 32-bit picks", (long long)d->empty);
    MSSR_REQUIRE(d->T >= 0 && d->T <= TC_MAX_T, "token_control: history of %lld tokens", (long long)d->T);
    MSSR_REQUIRE(d->ngram >= 0 && d->ngram <= 64, "token_control: n-grams of %d (0 = none, up to 64)", d->ngram);
    MSSR_REQUIRE(!d->allowed || (d->states >= 1 && d->state_mode >= 0 && d->state_mode <= 2 &&
                                 (d->state_mode != 1 || d->states >= d->B) && (d->state_mode != 2 || d->state)),
                 "token_control: mask table of %lld states, mode %d", (long long)d->states, d->state_mode);
    const bool hist = d->history && d->T > 0;
    const TcShape s = tc_shape(d->B, d->V, d->T, d->ids != nullptr);
    MSSR_REQUIRE(d->B <= TC_MAX_GRID / s.chunks, "token_control: %lld rows in one call", (long long)d->B);
    MSSR_REQUIRE(!d->out || tc_apart(d), "token_control: the new logits overlap the old ones without taking their place");
    MSSR_REQUIRE(!d->bias || (d->bias_bs >= 0 && d->bias_bs <= TC_MAX_LD), "token_control: bias rows %lld apart", (long long)d->bias_bs);
    MSSR_REQUIRE(!d->out || !d->bias || tc_bias_apart(d), "token_control: the new logits overlap the bias");
    MSSR_REQUIRE(!d->ids || s.chunks == 1 ||
                     (d->scratch && d->scratch_bytes >= d->B * s.chunks * (int64_t)sizeof(unsigned long long)),
                 "token_control: scratch of %lld bytes is too small", (long long)d->scratch_bytes);
    TokenControlArgs a{};
    a.logits = d->logits; a.out = d->out; a.ld = d->ld; a.ldo = d->ldo; a.V = d->V;
    a.B = (int)d->B; a.chunk = s.chunk; a.chunks = s.chunks;
    a.history = hist ? d->history : nullptr; a.h_bs = d->h_bs; a.h_ts = d->h_ts; a.h64 = d->index_bits & 1; a.T = d->T;
    a.lengths = {d->lengths, (d->index_bits >> 1) & 1, d->T};
    a.prompt = {d->prompt_lengths, (d->index_bits >> 2) & 1, 0};
    a.repetition = d->repetition; a.frequency = d->frequency; a.presence = d->presence;
    a.repetition0 = d->repetition0; a.frequency0 = d->frequency0; a.presence0 = d->presence0;
    a.ngram = d->ngram; a.bias = d->bias; a.bias_bs = d->bias_bs;
    a.allowed = (const uint32_t*)d->allowed; a.states = d->states; a.words = (d->V + 31) / 32;
    a.state = {d->state, (d->index_bits >> 3) & 1, 0}; a.state_mode = d->state_mode;
    a.ids = d->ids; a.ids64 = (d->index_bits >> 4) & 1; a.empty = d->empty;
    a.part = (unsigned long long*)d->scratch;
    const unsigned lds = hist ? (unsigned)s.chunk * (s.wide ? 4 : 2) : 0, grid = (unsigned)(d->B * s.chunks);
    hipStream_t st = (hipStream_t)stream;
    if (d->dtype == MSSR_F32) tc_launch<float>(a, s.wide, grid, lds, st);
    else tc_launch<bf16>(a, s.wide, grid, lds, st);
    if (d->ids && s.chunks > 1) token_pick_join_kernel<<<(unsigned)d->B, 64, 0, st>>>(a);
    MSSR_LAUNCH_OK("token_control");
}
