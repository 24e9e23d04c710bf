// Attention of a few new tokens over a 4-bit key/value cache (layout and numbers: kv4.hpp).
//
// With value = z + s * code per group g of 32 features,
//   q . k_t = sum_g s_tg (sum_{c in g} q_c code_tc) + z_tg (sum_{c in g} q_c)
//   o_c     = (sum_t (p_t s_tg) code_tc + sum_t p_t z_tg) / sum_t p_t
// so the matrix instructions take the CODES as they lie and the scales touch only scores and probabilities: one number
// a token instead of 32.  A code needs no conversion: the bit pattern of an integer c < 256 read as bf16 is the number
// c * 2^-133 (subnormals, which the matrix cores keep), so `x & 0x000f000f` IS an operand pair, `x & 0x00f000f0` one
// that is 16 times as large; the other operand carries 2^64 (q) or 2^96 (p s) so that every product is a normal fp32
// number, and powers of two cost nothing in precision.  8 codes take 5 vector instructions.
//
// A wave takes 64 tokens at a time, one token a lane from the scores on:
//   scores  4 products of 16 tokens x 32 features per group (mfma 16x16x32), accumulated into ONE result: the q operand
//           of product t is zero but for rows 4 t .. 4 t + 3, so lane (quad, n) ends with the scores of token
//           16 quad + n = its own number, for up to four query rows
//   softmax one token a lane; the running maximum moves only when a score passes it by more than 8 (then every sum is
//           rescaled), so that a block of tokens costs one comparison and no cross-lane reduction
//   p s     in bf16 parts (2 for bf16 queries: 2^-17 of p; 3 for fp32), transposed through 2 to 3 KB of LDS a group
//   context 2 products of 32 tokens per 16 features
// fp32 queries go in as three bf16 parts in three rows: one query row where bf16 ones have four.
#include "kv4.hpp"

namespace mssr {

struct Kv4AttnArgs {
    const uint8_t* data;
    int64_t blocks, capacity;
    const void* q;
    void* out;
    int64_t q_bs, q_hs, q_ts, o_bs, o_hs, o_ts;
    int Hkv, G, Tq, dh, causal;     // G query heads share a key/value head
    int NQ;                         // G * Tq query rows of a (sentence, key/value head)
    int splits;
    IdxTable lengths;
    float scale;                    // of the scores, times log2(e)
    float* part;                    // [rows][splits][dh] unnormalised context, then [rows][splits][2] (max, sum)
    int64_t rows;                   // B * Hkv * NQ
};

constexpr float KV4_QUP = 0x1p64f, KV4_PUP = 0x1p96f;
constexpr float KV4_SDOWN = 0x1p69f, KV4_ODOWN = 0x1p37f;      // 2^133 over the above

__device__ __forceinline__ float kv4_bf_lo(uint32_t w) { return __builtin_bit_cast(float, w << 16); }
__device__ __forceinline__ float kv4_bf_hi(uint32_t w) { return __builtin_bit_cast(float, w & 0xffff0000u); }
__device__ __forceinline__ uint16_t kv4_bf_bits(float x) { return __builtin_bit_cast(uint16_t, (bf16)x); }

// 8 codes of a K dword -> operand whose elements 2 r, 2 r + 1 are features 2 r, 2 r + 1 (r odd: times 16)
__device__ __forceinline__ bf16x8 kv4_k_operand(uint32_t x) {
    const uint32_t y = x >> 8;
    u32x4 r = {x & 0x000f000fu, x & 0x00f000f0u, y & 0x000f000fu, y & 0x00f000f0u};
    return __builtin_bit_cast(bf16x8, r);
}
// two V dwords (8 tokens) -> operands of feature n and of feature 16 + n (times 16); token order 0 2 1 3 4 6 5 7
__device__ __forceinline__ void kv4_v_operands(uint32_t x0, uint32_t x1, bf16x8& lo, bf16x8& hi) {
    const uint32_t y0 = x0 >> 8, y1 = x1 >> 8;
    u32x4 l = {x0 & 0x000f000fu, y0 & 0x000f000fu, x1 & 0x000f000fu, y1 & 0x000f000fu};
    u32x4 h = {x0 & 0x00f000f0u, y0 & 0x00f000f0u, x1 & 0x00f000f0u, y1 & 0x00f000f0u};
    lo = __builtin_bit_cast(bf16x8, l);
    hi = __builtin_bit_cast(bf16x8, h);
}

template <int NG>
struct Kv4Tile {            // a lane's share of a block: 16 NG bytes of K codes, of V codes, and its token's (s, z) pairs
    u32x4 k[NG], v[NG];
    uint32_t mk[NG], mv[NG];
    __device__ __forceinline__ void load(const uint8_t* blk, int lane) {
#pragma unroll
        for (int i = 0; i < NG; ++i) k[i] = *reinterpret_cast<const u32x4*>(blk + i * 1024 + lane * 16);
        __builtin_memcpy(mk, __builtin_assume_aligned(blk + NG * 2048 + lane * (4 * NG), 4), 4 * NG);
#pragma unroll
        for (int i = 0; i < NG; ++i) v[i] = *reinterpret_cast<const u32x4*>(blk + NG * 1024 + i * 1024 + lane * 16);
        __builtin_memcpy(mv, __builtin_assume_aligned(blk + NG * 2304 + lane * (4 * NG), 4), 4 * NG);
    }
};

// T: query type.  NG: groups of 32 features.  RS: row sets (of 4 bf16 query rows or 1 fp32 one) a block works on.
// W: waves; wave w takes every W-th block of the split.
template <typename T, int NG, int RS, int W>
__global__ __launch_bounds__(64 * W) void kv4_attention_kernel(Kv4AttnArgs a) {
    constexpr bool F32 = sizeof(T) == 4;
    constexpr int R = F32 ? 1 : 4;               // query rows of a row set
    constexpr int PARTS = F32 ? 3 : 2;           // bf16 parts of p s
    constexpr int PLD = 72;                      // bf16 elements of an LDS row of 64 tokens: 16-byte reads of 16 rows spread
    constexpr int DP = NG * 32;
    __shared__ __align__(16) uint16_t ps[W][NG * PARTS * 4][PLD];
    __shared__ float om[W > 1 ? W : 1][R][DP + 2];

    const int lane = threadIdx.x & 63, w = threadIdx.x >> 6, n = lane & 15, quad = lane >> 4;
    const int chunks = (a.NQ + RS * R - 1) / (RS * R);
    uint32_t id = blockIdx.x;
    const int split = id % a.splits;
    id /= a.splits;
    const int q0 = (int)(id % chunks) * (RS * R);
    const uint32_t bh = id / chunks;
    const int64_t b = bh / a.Hkv;
    const int hk = bh % a.Hkv;

    int64_t len = a.lengths.at(b);
    len = len < 0 ? 0 : (len > a.capacity ? a.capacity : len);
    const int64_t nb = (len + KV4_TOK - 1) / KV4_TOK, per = (nb + a.splits - 1) / a.splits;
    const int64_t first = split * per, last = first + per < nb ? first + per : nb;

    // query operands: lane (row n of the product, quad): features 32 g + 8 quad + 0..7 of query row 4 rs.. + (n & 3)
    bf16x8 qop[RS][NG];
    float qsum[RS][R][NG];                       // scale * sum of q over the group, every lane
    int64_t lim[RS][R];
    const T* qrow[RS][R];
    bool have[RS][R];
#pragma unroll
    for (int rs = 0; rs < RS; ++rs)
#pragma unroll
        for (int r = 0; r < R; ++r) {
            const int qi = q0 + rs * R + r;
            have[rs][r] = qi < a.NQ;
            const int i = have[rs][r] ? qi % a.Tq : 0, h = hk * a.G + (have[rs][r] ? qi / a.Tq : 0);
            qrow[rs][r] = (const T*)a.q + b * a.q_bs + h * a.q_hs + i * a.q_ts;
            lim[rs][r] = have[rs][r] ? (a.causal ? len - a.Tq + 1 + i : len) : 0;
        }
#pragma unroll
    for (int rs = 0; rs < RS; ++rs) {
#pragma unroll
        for (int g = 0; g < NG; ++g) {
            const int ch = g * 32 + quad * 8, r = F32 ? 0 : (n & 3);
            float x[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) x[e] = 0.f;
            const T* src = qrow[rs][0];
            bool on = have[rs][0];
            if (!F32) {
#pragma unroll
                for (int rr = 1; rr < R; ++rr)
                    if (r == rr) { src = qrow[rs][rr]; on = have[rs][rr]; }
            }
            if (on && ch < a.dh) {
                if constexpr (F32) {
                    __builtin_memcpy(x, src + ch, 32);
                } else {
                    bf16x8 v;
                    __builtin_memcpy(&v, src + ch, 16);
#pragma unroll
                    for (int e = 0; e < 8; ++e) x[e] = (float)v[e];
                }
            }
            float sum = ((x[0] + x[1]) + (x[2] + x[3])) + ((x[4] + x[5]) + (x[6] + x[7]));
            sum += __shfl_xor(sum, 16);
            sum += __shfl_xor(sum, 32);
#pragma unroll
            for (int rr = 0; rr < R; ++rr) qsum[rs][rr][g] = lane_read(sum, rr) * a.scale;
            bf16x8 op;
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                float y = x[e];
                if (F32) {                       // rows 0, 1, 2 of a quad: the three parts
                    const bf16 p0 = (bf16)y;
                    const float y1 = y - (float)p0;
                    const bf16 p1 = (bf16)y1;
                    const float y2 = y1 - (float)p1;
                    y = (n & 3) == 0 ? (float)p0 : (n & 3) == 1 ? (float)p1 : (n & 3) == 2 ? y2 : 0.f;
                }
                op[e] = (bf16)(y * (((e >> 1) & 1) ? KV4_QUP / 16.f : KV4_QUP));
            }
            qop[rs][g] = op;
        }
    }

    float m[RS][R], l[RS][R], zs[RS][R][NG];
    f32x4 acc[RS][2 * NG];
#pragma unroll
    for (int rs = 0; rs < RS; ++rs) {
#pragma unroll
        for (int r = 0; r < R; ++r) {
            m[rs][r] = -INFINITY;
            l[rs][r] = 0.f;
#pragma unroll
            for (int g = 0; g < NG; ++g) zs[rs][r][g] = 0.f;
        }
#pragma unroll
        for (int c = 0; c < 2 * NG; ++c) acc[rs][c] = f32x4{0.f, 0.f, 0.f, 0.f};
    }
    const uint8_t* base = a.data + (int64_t)bh * a.blocks * kv4_block_bytes(NG);
    const bf16x8 zero8 = {};

    Kv4Tile<NG> cur, nxt;
    if (first + w < last) cur.load(base + (first + w) * kv4_block_bytes(NG), lane);
    for (int64_t blk = first + w; blk < last; blk += W) {
        const bool more = blk + W < last;
        if (more) nxt.load(base + (blk + W) * kv4_block_bytes(NG), lane);
        const int64_t tok = blk * KV4_TOK + lane;
        // ---- scores
        f32x4 sc[RS][NG];
#pragma unroll
        for (int rs = 0; rs < RS; ++rs)
#pragma unroll
            for (int g = 0; g < NG; ++g) sc[rs][g] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int t = 0; t < 4; ++t)
#pragma unroll
            for (int g = 0; g < NG; ++g) {
                const bf16x8 kop = kv4_k_operand(cur.k[(t * NG + g) >> 2][(t * NG + g) & 3]);
#pragma unroll
                for (int rs = 0; rs < RS; ++rs) {
                    const bf16x8 qt = (n >> 2) == t ? qop[rs][g] : zero8;
                    sc[rs][g] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(qt, kop, sc[rs][g], 0, 0, 0);
                }
            }
        float ksc[NG], kz[NG], vsc[NG], vz[NG];
#pragma unroll
        for (int g = 0; g < NG; ++g) {           // past the sentence's end the cache may hold anything
            const uint32_t mk = tok < len ? cur.mk[g] : 0u, mv = tok < len ? cur.mv[g] : 0u;
            ksc[g] = kv4_scale(mk) * (KV4_SDOWN * a.scale);
            kz[g] = kv4_zero(mk);
            vsc[g] = kv4_scale(mv) * KV4_PUP;
            vz[g] = kv4_zero(mv);
        }
        bf16x8 vop[2][2 * NG];
#pragma unroll
        for (int ks = 0; ks < 2; ++ks)
#pragma unroll
            for (int g = 0; g < NG; ++g) {
                const int d = (ks * NG + g) * 2;
                kv4_v_operands(cur.v[d >> 2][d & 3], cur.v[d >> 2][(d & 3) + 1], vop[ks][2 * g], vop[ks][2 * g + 1]);
            }
#pragma unroll
        for (int rs = 0; rs < RS; ++rs) {
#pragma unroll
            for (int r = 0; r < R; ++r) {
                float s = 0.f;
#pragma unroll
                for (int g = 0; g < NG; ++g) {
                    const float dot = F32 ? sc[rs][g][0] + (sc[rs][g][1] + sc[rs][g][2]) : sc[rs][g][r];
                    s = fmaf(dot, ksc[g], s);
                    s = fmaf(qsum[rs][r][g], kz[g], s);
                }
                const bool see = tok < lim[rs][r];
                s = see ? s : -INFINITY;
                if (__any(s > m[rs][r] + 8.f)) {
                    const float mn = wave_max(s), f = __builtin_amdgcn_exp2f(m[rs][r] - mn);
                    m[rs][r] = mn;
                    l[rs][r] *= f;
#pragma unroll
                    for (int g = 0; g < NG; ++g) zs[rs][r][g] *= f;
#pragma unroll
                    for (int c = 0; c < 2 * NG; ++c) {
                        if (F32) acc[rs][c] *= f;
                        else acc[rs][c][r] *= f;
                    }
                }
                const float p = see ? __builtin_amdgcn_exp2f(s - m[rs][r]) : 0.f;
                l[rs][r] += p;
#pragma unroll
                for (int g = 0; g < NG; ++g) {
                    float y = see ? p * vsc[g] : 0.f;
                    zs[rs][r][g] += see ? p * vz[g] : 0.f;
                    // tokens 1 and 2 of four change places: the order of kv4_v_operands
                    const int col = (lane & ~3) | ((lane & 1) << 1) | ((lane >> 1) & 1);
#pragma unroll
                    for (int part = 0; part < PARTS; ++part) {
                        const bf16 h = (bf16)y;
                        y -= (float)h;
                        ps[w][(g * PARTS + part) * 4 + r][col] = __builtin_bit_cast(uint16_t, h);
                    }
                }
            }
            __builtin_amdgcn_wave_barrier();
            // ---- context: row 4 part + r of the product; rows of absent parts repeat others and are not used
#pragma unroll
            for (int ks = 0; ks < 2; ++ks)
#pragma unroll
                for (int g = 0; g < NG; ++g) {
                    const int row = (n >> 2) < PARTS ? n : (n & 3);
                    const u32x4 raw = *reinterpret_cast<const u32x4*>(&ps[w][g * PARTS * 4 + row][ks * 32 + quad * 8]);
                    const bf16x8 pop = __builtin_bit_cast(bf16x8, raw);
                    acc[rs][2 * g] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(pop, vop[ks][2 * g], acc[rs][2 * g], 0, 0, 0);
                    acc[rs][2 * g + 1] =
                        __builtin_amdgcn_mfma_f32_16x16x32_bf16(pop, vop[ks][2 * g + 1], acc[rs][2 * g + 1], 0, 0, 0);
                }
            __builtin_amdgcn_wave_barrier();
        }
        if (more) cur = nxt;
    }

    // ---- sums over lanes, then over the block's waves
#pragma unroll
    for (int rs = 0; rs < RS; ++rs) {
        if (W > 1 && rs) __syncthreads();
#pragma unroll
        for (int r = 0; r < R; ++r) {
            const float lt = wave_sum(l[rs][r]);
            float zt[NG];
#pragma unroll
            for (int g = 0; g < NG; ++g) zt[g] = wave_sum(zs[rs][r][g]);
#pragma unroll
            for (int c = 0; c < 2 * NG; ++c) {
                float v = acc[rs][c][r];
                float u = v + __shfl_xor(v, 16);                    // parts 0 + 1 (quads 0 and 1)
                if (PARTS == 3) u += __shfl_xor(v, 32);             // quad 0: + part 2
                u = fmaf(u, (c & 1) ? KV4_ODOWN / 16.f : KV4_ODOWN, zt[c >> 1]);
                if (quad == 0) om[w][r][c * 16 + n] = u;
            }
            if (lane == 0) {
                om[w][r][DP] = m[rs][r];
                om[w][r][DP + 1] = lt;
            }
        }
        if (W > 1) __syncthreads();
        else __builtin_amdgcn_wave_barrier();
        for (int x = threadIdx.x; x < R * DP; x += 64 * W) {
            const int r = x / DP, c = x % DP, qi = q0 + rs * R + r;
            if (qi >= a.NQ || c >= a.dh) continue;
            float top = om[0][r][DP], sum = 0.f, o = 0.f;
#pragma unroll
            for (int k = 1; k < W; ++k) top = fmaxf(top, om[k][r][DP]);
#pragma unroll
            for (int k = 0; k < W; ++k) {
                const float mk = om[k][r][DP];
                // a wave that saw nothing has nothing to add (and its maximum is minus infinity)
                const float f = mk == -INFINITY && om[k][r][DP + 1] == 0.f ? 0.f : __builtin_amdgcn_exp2f(mk - top);
                sum = fmaf(f, om[k][r][DP + 1], sum);
                o = fmaf(f, om[k][r][c], o);
            }
            if (a.splits == 1) {
                const int i = qi % a.Tq, h = hk * a.G + qi / a.Tq;
                ((T*)a.out)[b * a.o_bs + h * a.o_hs + i * a.o_ts + c] = from_f<T>(sum == 0.f ? 0.f : o / sum);
            } else {
                const int64_t row = (int64_t)bh * a.NQ + qi, at = row * a.splits + split;
                a.part[at * a.dh + c] = o;
                if (c == 0) {
                    float* ml = a.part + a.rows * a.splits * a.dh + at * 2;
                    ml[0] = top;
                    ml[1] = sum;
                }
            }
        }
    }
}

// joins the splits of a query row: one wave a row
template <typename T>
__global__ __launch_bounds__(64) void kv4_join_kernel(Kv4AttnArgs a) {
    const int64_t row = blockIdx.x;
    const float* ml = a.part + a.rows * a.splits * a.dh + row * a.splits * 2;
    float top = -INFINITY;
    for (int s = threadIdx.x; s < a.splits; s += 64) top = fmaxf(top, ml[2 * s]);
    top = wave_max(top);
    float sum = 0.f, o0 = 0.f, o1 = 0.f;
    const int c0 = threadIdx.x, c1 = c0 + 64;
    const float* o = a.part + row * a.splits * a.dh;
    for (int s = 0; s < a.splits; ++s) {
        const float m = ml[2 * s], l = ml[2 * s + 1];
        const float f = m == -INFINITY && l == 0.f ? 0.f : __builtin_amdgcn_exp2f(m - top);
        sum = fmaf(f, l, sum);
        if (c0 < a.dh) o0 = fmaf(f, o[(int64_t)s * a.dh + c0], o0);
        if (c1 < a.dh) o1 = fmaf(f, o[(int64_t)s * a.dh + c1], o1);
    }
    const int64_t bh = row / a.NQ;
    const int qi = (int)(row % a.NQ), i = qi % a.Tq;
    const int64_t b = bh / a.Hkv, h = (bh % a.Hkv) * a.G + qi / a.Tq;
    T* dst = (T*)a.out + b * a.o_bs + h * a.o_hs + i * a.o_ts;
    if (c0 < a.dh) dst[c0] = from_f<T>(sum == 0.f ? 0.f : o0 / sum);
    if (c1 < a.dh) dst[c1] = from_f<T>(sum == 0.f ? 0.f : o1 / sum);
}

struct Kv4Shape { int RS, W, splits; int64_t units, chunks; };

// How a call is cut: `longest` bounds the lengths (the capacity where the caller knows no better).
static Kv4Shape kv4_shape(int64_t B, int Hkv, int NQ, int dtype, int64_t longest) {
    Kv4Shape s;
    const int R = dtype == MSSR_F32 ? 1 : 4;
    s.RS = NQ > R ? 2 : 1;
    s.chunks = (NQ + s.RS * R - 1) / (s.RS * R);
    s.units = B * Hkv * s.chunks;
    const int64_t nb = (longest + KV4_TOK - 1) / KV4_TOK;
    s.W = nb <= 1 || s.units >= 4096 ? 1 : 4;
    const int64_t want = 4096 / (s.units * s.W), most = (nb + s.W - 1) / s.W;
    s.splits = (int)(want < 1 ? 1 : (want > most ? most : want));
    if (s.splits > 512) s.splits = 512;
    return s;
}

template <typename T, int NG, int RS>
static void kv4_launch(const Kv4AttnArgs& a, const Kv4Shape& s, hipStream_t st) {
    const unsigned grid = (unsigned)(s.units * s.splits);
    if (s.W == 1) kv4_attention_kernel<T, NG, RS, 1><<<grid, 64, 0, st>>>(a);
    else kv4_attention_kernel<T, NG, RS, 4><<<grid, 256, 0, st>>>(a);
}
template <typename T>
static void kv4_dispatch(const Kv4AttnArgs& a, const Kv4Shape& s, int ng, hipStream_t st) {
#define MSSR_KV4_A(NG)                                  \
    case NG:                                            \
        if (s.RS == 1) kv4_launch<T, NG, 1>(a, s, st);  \
        else kv4_launch<T, NG, 2>(a, s, st);            \
        break;
    switch (ng) { MSSR_KV4_A(1) MSSR_KV4_A(2) MSSR_KV4_A(3) MSSR_KV4_A(4) }
#undef MSSR_KV4_A
    if (a.splits > 1) kv4_join_kernel<T><<<(unsigned)a.rows, 64, 0, st>>>(a);
}

}  // namespace mssr

using namespace mssr;

static int64_t kv4_longest(const mssr_kv4_cache* c, int64_t longest) {
    return longest < 1 || longest > c->capacity ? c->capacity : longest;
}

extern "C" int64_t mssr_kv4_attention_scratch(const mssr_kv4_cache* c, int64_t Tq, int H, int64_t longest, int dtype) {
    if (!c || c->B < 1 || c->H < 1 || H < c->H || H % c->H || Tq < 1 || c->capacity < 1 || !valid_dtype(dtype)) return -1;
    if (Tq > INT32_MAX / (H / c->H)) return -1;
    const int NQ = (int)(H / c->H * Tq);
    const Kv4Shape s = kv4_shape(c->B, c->H, NQ, dtype, kv4_longest(c, longest));
    return s.splits > 1 ? c->B * c->H * NQ * s.splits * (c->dh + 2) * (int64_t)sizeof(float) : 0;
}

extern "C" int mssr_kv4_attention(const mssr_kv4_cache* c, const void* q, int64_t q_bs, int64_t q_hs, int64_t q_ts, void* out,
                                  int64_t o_bs, int64_t o_hs, int64_t o_ts, int H, int64_t Tq, const void* lengths,
                                  int64_t length0, int lengths_are_64, int64_t longest, float scale, int causal, void* scratch,
                                  int64_t scratch_bytes, int dtype, void* stream) {
    MSSR_REQUIRE(c && c->data && (Tq == 0 || (q && out)), "kv4_attention: null operand");
    MSSR_REQUIRE(mssr_kv4_bytes(c->B, c->H, c->capacity, c->dh) > 0 && aligned(c->data, 16),
                 "kv4_attention: cache of %lld x %d heads x %lld tokens x %d features (multiples of 8 up to %d)",
                 (long long)c->B, c->H, (long long)c->capacity, c->dh, KV4_MAX_DH);
    MSSR_REQUIRE(valid_dtype(dtype), "kv4_attention: dtype %d", dtype);
    MSSR_REQUIRE(Tq >= 0 && H >= c->H && H % c->H == 0, "kv4_attention: %d query heads on %d, %lld rows", H, c->H, (long long)Tq);
    MSSR_REQUIRE(lengths || (length0 >= 0 && length0 <= c->capacity), "kv4_attention: length %lld of a cache of %lld",
                 (long long)length0, (long long)c->capacity);
    if (Tq == 0) return MSSR_OK;
    MSSR_REQUIRE(Tq <= (INT32_MAX >> 8) / (H / c->H), "kv4_attention: %lld query rows", (long long)Tq);
    const int NQ = (int)(H / c->H * Tq);
    const Kv4Shape s = kv4_shape(c->B, c->H, NQ, dtype, kv4_longest(c, longest));
    const int64_t rows = c->B * c->H * NQ;
    MSSR_REQUIRE(s.units <= KV4_MAX_GRID / s.splits && rows <= KV4_MAX_GRID, "kv4_attention: %lld query rows in one call",
                 (long long)rows);
    MSSR_REQUIRE(s.splits == 1 || (scratch && scratch_bytes >= rows * s.splits * (c->dh + 2) * (int64_t)sizeof(float)),
                 "kv4_attention: scratch of %lld bytes is too small", (long long)scratch_bytes);
    Kv4AttnArgs a{(const uint8_t*)c->data, (c->capacity + KV4_TOK - 1) / KV4_TOK, c->capacity, q, out, q_bs, q_hs, q_ts,
                  o_bs, o_hs, o_ts, c->H, H / c->H, (int)Tq, c->dh, causal ? 1 : 0, NQ, s.splits,
                  {lengths, lengths_are_64, length0}, scale * 1.4426950408889634f, (float*)scratch, rows};
    if (dtype == MSSR_F32) kv4_dispatch<float>(a, s, kv4_groups(c->dh), (hipStream_t)stream);
    else kv4_dispatch<bf16>(a, s, kv4_groups(c->dh), (hipStream_t)stream);
    MSSR_LAUNCH_OK("kv4_attention");
}
