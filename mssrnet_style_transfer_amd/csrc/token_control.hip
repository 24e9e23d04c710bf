// Control of the next token's logits: penalties for tokens of the history, a bias, a grammar's mask, no repeated n-grams;
// either the new logits or only the pick (the largest) leaves.
//
// Per row, in fp32 with every step rounded:
//   v in the history:  x = x > 0 ? x / repetition : x * repetition
//   x = x - (frequency * count + presence * (count > 0)),  count over the history from prompt_lengths on
//   x = x + bias[v];   x = -inf where the mask's bit is 0 or v would complete an n-gram of the history
// Bound by memory: the logits once, written once or not at all.  A block owns a chunk of a row: it walks the history
// first and keeps, for the chunk's words, one LDS word each (count, seen, banned), then streams the logits.  Few rows
// are cut into many chunks (their picks are joined by a second launch), many rows into few.
#include "common.hpp"
#include "kv4.hpp"      // IdxTable

namespace mssr {

constexpr uint32_t TC_SEEN = 0x80000000u, TC_BANNED = 0x40000000u, TC_COUNT = 0x3fffffffu;
constexpr int TC_UNIT = 2048;                    // a chunk is a multiple of 256 threads x 8 words
constexpr int TC_MAX_CHUNK = 16384;              // 64 KB of LDS words

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

template <typename T>
__global__ __launch_bounds__(256) void token_control_kernel(TokenControlArgs a) {
#pragma clang fp contract(off)
    extern __shared__ uint32_t mark[];
    __shared__ unsigned long long best[4];
    const int64_t b = blockIdx.x / (uint32_t)a.chunks;
    const int ci = blockIdx.x % (uint32_t)a.chunks;
    const int64_t v0 = (int64_t)ci * a.chunk;
    const int n = (int)(a.V - v0 < a.chunk ? a.V - v0 : a.chunk);
    const float rep = a.repetition ? a.repetition[b] : a.repetition0;
    const float freq = a.frequency ? a.frequency[b] : a.frequency0;
    const float pres = a.presence ? a.presence[b] : a.presence0;

    if (a.history) {
        int64_t len = a.lengths.p ? a.lengths.at(b) : a.T;
        len = len < 0 ? 0 : (len > a.T ? a.T : len);
        const int64_t from = a.prompt.at(b);
        for (int i = threadIdx.x; i < n; i += 256) mark[i] = 0;
        __syncthreads();
        for (int64_t t = threadIdx.x; t < len; t += 256) {
            const int64_t at = tc_token(a, b, t) - v0;
            if (at < 0 || at >= n) continue;
            if (t >= from) atomicAdd(&mark[at], 1u);
            uint32_t flags = TC_SEEN;
            if (a.ngram == 1) flags |= TC_BANNED;
            if (a.ngram > 1 && t >= a.ngram - 1) {
                bool same = true;
                for (int j = 1; j < a.ngram && same; ++j) same = tc_token(a, b, t - j) == tc_token(a, b, len - j);
                if (same) flags |= TC_BANNED;
            }
            atomicOr(&mark[at], flags);
        }
        __syncthreads();
    }
    const uint32_t* mask = nullptr;
    bool closed = false;
    if (a.allowed) {
        const int64_t st = a.state_mode == 0 ? 0 : a.state_mode == 1 ? b : a.state.at(b);
        if (st >= a.states) closed = true;       // not a state of the table: nothing is allowed
        else if (st >= 0) mask = a.allowed + st * a.words;
    }
    const T* x = (const T*)a.logits + b * a.ld + v0;
    const float* bias = a.bias ? a.bias + b * a.bias_bs + v0 : nullptr;
    unsigned long long top = 0;
    for (int i = threadIdx.x; i < n; i += 256) {
        float y = to_f(x[i]);
        bool banned = closed;
        if (a.history) {
            const uint32_t mk = mark[i];
            if (mk) {
                y = y > 0.f ? y / rep : y * rep;
                const uint32_t c = mk & TC_COUNT;
                y = y - (freq * (float)c + (c ? pres : 0.f));
                banned |= (mk & TC_BANNED) != 0;
            }
        }
        if (bias) y = y + bias[i];
        const int64_t v = v0 + i;
        if (mask) banned |= !((mask[v >> 5] >> (v & 31)) & 1u);
        if (banned) y = -INFINITY;
        if (a.out) ((T*)a.out)[b * a.ldo + v] = from_f<T>(y);
        if (a.ids) {
            const unsigned long long k = tc_key(y, (uint32_t)v);
            top = k > top ? k : top;
        }
    }
    if (!a.ids) return;
    top = tc_wave_max(top);
    if ((threadIdx.x & 63) == 0) best[threadIdx.x >> 6] = top;
    __syncthreads();
    if (threadIdx.x) return;
    for (int w = 1; w < 4; ++w) top = best[w] > top ? best[w] : top;
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

struct TcShape { int chunk, chunks; };
static TcShape tc_shape(int64_t B, int64_t V) {
    const int64_t least = (V + TC_MAX_CHUNK - 1) / TC_MAX_CHUNK, most = (V + TC_UNIT - 1) / TC_UNIT;
    int64_t c = (1024 + B - 1) / B;
    c = c < least ? least : (c > most ? most : c);
    TcShape s;
    s.chunk = (int)(((V + c - 1) / c + TC_UNIT - 1) / TC_UNIT * TC_UNIT);
    s.chunks = (int)((V + s.chunk - 1) / s.chunk);
    return s;
}

}  // namespace mssr

using namespace mssr;

extern "C" int64_t mssr_token_control_scratch(int64_t B, int64_t V) {
    if (B < 1 || V < 1 || V > INT32_MAX) return -1;
    const TcShape s = tc_shape(B, V);
    return s.chunks > 1 ? B * s.chunks * (int64_t)sizeof(unsigned long long) : 0;
}

extern "C" int mssr_token_control(const mssr_token_control_desc* d, void* stream) {
    MSSR_REQUIRE(d, "token_control: no descriptor");
    MSSR_REQUIRE(d->B >= 0 && d->V >= 1 && d->V <= INT32_MAX && d->ld >= d->V, "token_control: logits [%lld, %lld], row stride %lld",
                 (long long)d->B, (long long)d->V, (long long)d->ld);
    MSSR_REQUIRE(valid_dtype(d->dtype), "token_control: dtype %d", d->dtype);
    if (d->B == 0) return MSSR_OK;
    MSSR_REQUIRE(d->logits && (d->out || d->ids), "token_control: null operand");
    MSSR_REQUIRE(!d->out || d->ldo >= d->V, "token_control: row stride %lld of the new logits", (long long)d->ldo);
    MSSR_REQUIRE(d->T >= 0 && d->T <= TC_COUNT, "token_control: history of %lld tokens", (long long)d->T);
    MSSR_REQUIRE(d->ngram >= 0 && d->ngram <= 64, "token_control: n-grams of %d (0 = none, up to 64)", d->ngram);
    MSSR_REQUIRE(!d->allowed || (d->states >= 1 && d->state_mode >= 0 && d->state_mode <= 2 &&
                                 (d->state_mode != 1 || d->states >= d->B) && (d->state_mode != 2 || d->state)),
                 "token_control: mask table of %lld states, mode %d", (long long)d->states, d->state_mode);
    const TcShape s = tc_shape(d->B, d->V);
    MSSR_REQUIRE(d->B <= KV4_MAX_GRID / s.chunks, "token_control: %lld rows in one call", (long long)d->B);
    MSSR_REQUIRE(!d->ids || s.chunks == 1 ||
                     (d->scratch && d->scratch_bytes >= d->B * s.chunks * (int64_t)sizeof(unsigned long long)),
                 "token_control: scratch of %lld bytes is too small", (long long)d->scratch_bytes);
    const bool hist = d->history && d->T > 0;
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
    const unsigned lds = hist ? (unsigned)s.chunk * 4 : 0;
    const unsigned grid = (unsigned)(d->B * s.chunks);
    hipStream_t st = (hipStream_t)stream;
    if (d->dtype == MSSR_F32) token_control_kernel<float><<<grid, 256, lds, st>>>(a);
    else token_control_kernel<bf16><<<grid, 256, lds, st>>>(a);
    if (d->ids && s.chunks > 1) token_pick_join_kernel<<<(unsigned)d->B, 64, 0, st>>>(a);
    MSSR_LAUNCH_OK("token_control");
}
