// Attention of a few new tokens over a 4-bit key/value cache (layout and numbers: kv4.hpp).
//
// With value = z + s * code per group g of 32 features,
//   q . k_t = sum_g s_tg (sum_{c in g} q_c code_tc) + z_tg (sum_{c in g} q_c)
//   o_c     = (sum_t (p_t s_tg) code_tc + sum_t p_t z_tg) / sum_t p_t
// so the matrix instructions take the CODES as they lie and the scales touch only scores and probabilities: one number
// a token instead of 32.  A code needs no conversion: the bit pattern of an integer c < 256 read as bf16 is the number
// c * 2^-133 (subnormals, which the matrix cores keep), so `x & 0x000f000f` IS an operand pair, `x & 0x00f000f0` one
// that is 16 times as large; the other operand (q, or p s) carries 2^64 so that every product is a normal fp32 number,
// and powers of two cost nothing in precision.  8 codes take 5 vector instructions.
//
// A number enters a product as bf16 parts whose products add up in fp32: bf16 queries are one part, fp32 ones three (all
// 24 bits); p s, an fp32 number, two for bf16 results (2^-17 of it is lost, 2^-8 of the result is rounded away) and three
// for fp32 ones.
//
// A wave takes 64 tokens at a time; the running maximum moves only when a score passes it by more than 8 (then every
// sum is rescaled), so that a block of tokens costs one comparison and no cross-lane reduction.  The W waves of a block
// take every W-th 64 tokens of its share of the sentence and are joined through LDS; a second launch joins the shares.
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

constexpr float KV4_UP = 0x1p64f, KV4_DOWN = 0x1p69f;          // UP * DOWN * 2^-133 = 1
constexpr float KV4_LAZY = 8.f;                                // log2 of how far a probability may pass 1 before a rescale
constexpr int KV4_UPLOG = 64;

// 8 codes of a K dword -> operand whose elements 2 r, 2 r + 1 are features 2 r, 2 r + 1 (r odd: times 16)
__device__ __forceinline__ bf16x8 kv4_k_operand(uint32_t x) {
    const uint32_t y = x >> 8;
    u32x4 r = {x & 0x000f000fu, x & 0x00f000f0u, y & 0x000f000fu, y & 0x00f000f0u};
    return __builtin_bit_cast(bf16x8, r);
}
// two V dwords (4 tokens of tile 2 ks, 4 of tile 2 ks + 1) -> operands of feature n and of feature 16 + n (times 16);
// the four tokens of a dword come in the order 0 2 1 3
__device__ __forceinline__ void kv4_v_operands(uint32_t x0, uint32_t x1, bf16x8& lo, bf16x8& hi) {
    const uint32_t y0 = x0 >> 8, y1 = x1 >> 8;
    u32x4 l = {x0 & 0x000f000fu, y0 & 0x000f000fu, x1 & 0x000f000fu, y1 & 0x000f000fu};
    u32x4 h = {x0 & 0x00f000f0u, y0 & 0x00f000f0u, x1 & 0x00f000f0u, y1 & 0x00f000f0u};
    lo = __builtin_bit_cast(bf16x8, l);
    hi = __builtin_bit_cast(bf16x8, h);
}
__device__ __forceinline__ f32x4 kv4_mfma(bf16x8 a, bf16x8 b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
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

struct Kv4Work {            // what a block works on: query rows q0 .. of (sentence, key/value head), blocks [first, last)
    int64_t b, bh, len, first, last;
    int hk, q0, split;
    __device__ __forceinline__ Kv4Work(const Kv4AttnArgs& a, int rows) {
        const uint32_t chunks = (a.NQ + rows - 1) / rows;
        uint32_t id = blockIdx.x;
        split = id % a.splits;
        id /= a.splits;
        q0 = (int)(id % chunks) * rows;
        bh = id / chunks;
        b = bh / a.Hkv;
        hk = (int)(bh % a.Hkv);
        len = a.lengths.at(b);
        len = len < 0 ? 0 : (len > a.capacity ? a.capacity : len);
        const int64_t nb = (len + KV4_TOK - 1) / KV4_TOK, per = (nb + a.splits - 1) / a.splits;
        first = split * per;
        last = first + per < nb ? first + per : nb;
    }
};

// 8 features of a query row as bf16 parts times 2^64 (elements that meet a code times 16: 2^60); returns their sum
template <typename T, int PARTS>
__device__ __forceinline__ float kv4_query(const T* src, bool on, bf16x8 (&op)[PARTS]) {
    float x[8] = {};
    if (on) {
        if constexpr (sizeof(T) == 4) {
            __builtin_memcpy(x, src, 32);
        } else {
            bf16x8 v;
            __builtin_memcpy(&v, src, 16);
#pragma unroll
            for (int e = 0; e < 8; ++e) x[e] = (float)v[e];
        }
    }
    const float sum = ((x[0] + x[1]) + (x[2] + x[3])) + ((x[4] + x[5]) + (x[6] + x[7]));
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        float y = x[e];
#pragma unroll
        for (int p = 0; p < PARTS; ++p) {
            const bf16 h = (bf16)y;
            y -= (float)h;
            op[p][e] = (bf16)((float)h * (((e >> 1) & 1) ? KV4_UP / 16.f : KV4_UP));
        }
    }
    return sum;
}

// Joins the block's waves (om: per wave and row the context, maximum and sum; synchronised by the caller) and writes the
// row, or its share of it.
template <typename T, int W, int R, int DP>
__device__ __forceinline__ void kv4_finish(const Kv4AttnArgs& a, const Kv4Work& wk, const float (&om)[W][R][DP + 4]) {
    for (int x = threadIdx.x; x < R * (DP / 2); x += 64 * W) {
        const int r = x / (DP / 2), c = x % (DP / 2) * 2, qi = wk.q0 + r;
        if (qi >= a.NQ || c >= a.dh) continue;
        float top = om[0][r][DP], sum = 0.f, o0 = 0.f, o1 = 0.f;
#pragma unroll
        for (int k = 1; k < W; ++k) top = fmaxf(top, om[k][r][DP]);
#pragma unroll
        for (int k = 0; k < W; ++k) {
            const float mk = om[k][r][DP], lk = om[k][r][DP + 1];
            // a wave that saw nothing has nothing to add (its maximum is minus infinity, like the joint one may be)
            const float f = mk == -INFINITY && lk == 0.f ? 0.f : __builtin_amdgcn_exp2f(mk - top);
            sum = fmaf(f, lk, sum);
            o0 = fmaf(f, om[k][r][c], o0);
            o1 = fmaf(f, om[k][r][c + 1], o1);
        }
        if (a.splits == 1) {
            const int i = qi % a.Tq, h = wk.hk * a.G + qi / a.Tq;
            T* dst = (T*)a.out + wk.b * a.o_bs + h * a.o_hs + i * a.o_ts + c;
            dst[0] = from_f<T>(sum == 0.f ? 0.f : o0 / sum);
            dst[1] = from_f<T>(sum == 0.f ? 0.f : o1 / sum);
        } else {
            const int64_t at = (wk.bh * a.NQ + qi) * a.splits + wk.split;
            a.part[at * a.dh + c] = o0;
            a.part[at * a.dh + c + 1] = o1;
            if (c == 0) {
                float* ml = a.part + a.rows * a.splits * a.dh + at * 2;
                ml[0] = top;
                ml[1] = sum;
            }
        }
    }
}

// Up to 4 query rows (R of them in use) of a key/value head: the decode step.  One token a lane from the scores on.
//   scores   per group 4 products of 16 tokens; every quad of rows of the q operand holds the same rows, so lane
//            (quad, n) finds token n of each product and keeps the one of its own 16 (one fp32 row: its 3 parts are rows)
//   p s      goes through LDS to become an operand: row 4 part + r, the parts add up at the end
// Bound by the cache's bytes: at 64 features about 130 vector and 16 matrix instructions for 5 KB.
template <typename T, int NG, int R, int W>
__global__ __launch_bounds__(64 * W) void kv4_few_kernel(Kv4AttnArgs a) {
    constexpr bool F32 = sizeof(T) == 4;
    constexpr bool QROWS = F32 && R == 1;        // the parts of q in rows of one product instead of products of their own
    constexpr int QP = F32 ? 3 : 1, PP = F32 ? 3 : 2;
    constexpr int PLD = 72;                      // bf16 elements of an LDS row of 64 tokens: 16-byte reads of 16 rows spread
    constexpr int DP = NG * 32;
    __shared__ __align__(16) uint16_t ps[W][NG][PP * R][PLD];
    __shared__ float om[W][R][DP + 4];

    const int lane = threadIdx.x & 63, w = threadIdx.x >> 6, n = lane & 15, quad = lane >> 4;
    const Kv4Work wk(a, R);
    bf16x8 qop[QROWS ? 1 : QP][NG];
    float qsum[R][NG];                           // scale * sum of q over the group
    int64_t lim[R];
    {
        const int r = R == 1 ? 0 : (n & 3), qi = wk.q0 + r;
        const bool have = qi < a.NQ;
        const int i = have ? qi % a.Tq : 0, h = wk.hk * a.G + (have ? qi / a.Tq : 0);
        const T* src = (const T*)a.q + wk.b * a.q_bs + h * a.q_hs + i * a.q_ts;
#pragma unroll
        for (int g = 0; g < NG; ++g) {
            const int ch = g * 32 + quad * 8;
            bf16x8 op[QP];
            float sum = kv4_query<T, QP>(src + ch, have && ch < a.dh, op);
            sum += __shfl_xor(sum, 16);
            sum += __shfl_xor(sum, 32);
#pragma unroll
            for (int rr = 0; rr < R; ++rr) qsum[rr][g] = lane_read(sum, rr) * a.scale;
            if constexpr (QROWS) {
                const bf16x8 none = {};
                qop[0][g] = (n & 3) == 0 ? op[0] : (n & 3) == 1 ? op[1] : (n & 3) == 2 ? op[2] : none;
            } else {
#pragma unroll
                for (int p = 0; p < QP; ++p) qop[p][g] = op[p];
            }
        }
#pragma unroll
        for (int rr = 0; rr < R; ++rr) {
            const int k = wk.q0 + rr;
            lim[rr] = k < a.NQ ? (a.causal ? wk.len - a.Tq + 1 + k % a.Tq : wk.len) : 0;
        }
    }

    float m[R], l[R], zs[R][NG];                 // m: the reference of the exponents, 64 below the running maximum's
    f32x4 acc[2 * NG];
#pragma unroll
    for (int r = 0; r < R; ++r) {
        m[r] = -INFINITY;
        l[r] = 0.f;
#pragma unroll
        for (int g = 0; g < NG; ++g) zs[r][g] = 0.f;
    }
#pragma unroll
    for (int c = 0; c < 2 * NG; ++c) acc[c] = f32x4{0.f, 0.f, 0.f, 0.f};
    const uint8_t* base = a.data + wk.bh * a.blocks * kv4_block_bytes(NG);
    const float down = KV4_DOWN * a.scale;
    // where this lane's token goes among the operand's 64: half, quad, then 0 2 1 3
    const int col = (lane & 32) | ((lane & 12) << 1) | ((lane & 16) >> 2) | ((lane & 1) << 1) | ((lane >> 1) & 1);
    const f32x4 zero4 = {0.f, 0.f, 0.f, 0.f};

    Kv4Tile<NG> cur, nxt;
    if (wk.first + w < wk.last) cur.load(base + (wk.first + w) * kv4_block_bytes(NG), lane);
    for (int64_t blk = wk.first + w; blk < wk.last; blk += W) {
        const bool more = blk + W < wk.last;
        if (more) nxt.load(base + (blk + W) * kv4_block_bytes(NG), lane);
        const int64_t tok = blk * KV4_TOK + lane;
        uint32_t mk[NG], mv[NG];
#pragma unroll
        for (int g = 0; g < NG; ++g) {           // past the sentence's end the cache may hold anything
            mk[g] = tok < wk.len ? cur.mk[g] : 0u;
            mv[g] = tok < wk.len ? cur.mv[g] : 0u;
        }
        float dot[R], off[R];
#pragma unroll
        for (int r = 0; r < R; ++r) dot[r] = off[r] = 0.f;
#pragma unroll
        for (int g = 0; g < NG; ++g) {
            f32x4 d[4];
#pragma unroll
            for (int t = 0; t < 4; ++t) {
                const bf16x8 kop = kv4_k_operand(cur.k[(t * NG + g) >> 2][(t * NG + g) & 3]);
                d[t] = kv4_mfma(qop[0][g], kop, zero4);
                if constexpr (!QROWS) {
#pragma unroll
                    for (int p = 1; p < QP; ++p) d[t] = kv4_mfma(qop[p][g], kop, d[t]);
                }
            }
#pragma unroll
            for (int r = 0; r < R; ++r) {
                float x = quad == 0 ? d[0][r] : quad == 1 ? d[1][r] : quad == 2 ? d[2][r] : d[3][r];
                if constexpr (QROWS) {
                    x += (quad == 0 ? d[0][1] : quad == 1 ? d[1][1] : quad == 2 ? d[2][1] : d[3][1]) +
                         (quad == 0 ? d[0][2] : quad == 1 ? d[1][2] : quad == 2 ? d[2][2] : d[3][2]);
                }
                dot[r] = fmaf(x, kv4_scale(mk[g]), dot[r]);
                off[r] = fmaf(qsum[r][g], kv4_zero(mk[g]), off[r]);
            }
        }
#pragma unroll
        for (int r = 0; r < R; ++r) {
            const bool see = tok < lim[r];
            const float s = see ? fmaf(dot[r], down, off[r]) : -INFINITY;
            if (__any(s - KV4_UPLOG > m[r] + KV4_LAZY)) {
                const float mn = wave_max(s) - KV4_UPLOG, f = __builtin_amdgcn_exp2f(m[r] - mn);
                m[r] = mn;
                l[r] *= f;
#pragma unroll
                for (int g = 0; g < NG; ++g) zs[r][g] *= f;
#pragma unroll
                for (int c = 0; c < 2 * NG; ++c) acc[c][r] *= f;
            }
            const float p = see ? __builtin_amdgcn_exp2f(s - m[r]) : 0.f;
            l[r] += p;
#pragma unroll
            for (int g = 0; g < NG; ++g) {
                float y = see ? p * kv4_scale(mv[g]) : 0.f;
                zs[r][g] += see ? p * kv4_zero(mv[g]) : 0.f;
#pragma unroll
                for (int part = 0; part < PP; ++part) {
                    const bf16 h = (bf16)y;
                    y -= (float)h;
                    ps[w][g][part * R + r][col] = __builtin_bit_cast(uint16_t, h);
                }
            }
        }
        __builtin_amdgcn_wave_barrier();
        // rows 4 part + r; the rows of absent parts and queries repeat others and are not used
        const int row = R == 1 ? ((n >> 2) < PP ? (n >> 2) : 0) : ((n >> 2) < PP ? n : (n & 3));
#pragma unroll
        for (int ks = 0; ks < 2; ++ks)
#pragma unroll
            for (int g = 0; g < NG; ++g) {
                const int d = (ks * NG + g) * 2;
                bf16x8 lo, hi;
                kv4_v_operands(cur.v[d >> 2][d & 3], cur.v[d >> 2][(d & 3) + 1], lo, hi);
                const u32x4 raw = *reinterpret_cast<const u32x4*>(&ps[w][g][row][ks * 32 + quad * 8]);
                const bf16x8 pop = __builtin_bit_cast(bf16x8, raw);
                acc[2 * g] = kv4_mfma(pop, lo, acc[2 * g]);
                acc[2 * g + 1] = kv4_mfma(pop, hi, acc[2 * g + 1]);
            }
        __builtin_amdgcn_wave_barrier();
        if (more) cur = nxt;
    }

#pragma unroll
    for (int r = 0; r < R; ++r) {
        const float lt = wave_sum(l[r]) * (1.f / KV4_UP);
        float zt[NG];
#pragma unroll
        for (int g = 0; g < NG; ++g) zt[g] = wave_sum(zs[r][g]) * (1.f / KV4_UP);
#pragma unroll
        for (int c = 0; c < 2 * NG; ++c) {
            const float v = acc[c][r];
            float u = v + __shfl_xor(v, 16);                    // parts 0 + 1 (quads 0 and 1)
            if (PP == 3) u += __shfl_xor(v, 32);                // quad 0: + part 2
            u = fmaf(u, (c & 1) ? KV4_DOWN / 16.f : KV4_DOWN, zt[c >> 1]);
            if (quad == 0) om[w][r][c * 16 + n] = u;
        }
        if (lane == 0) {
            om[w][r][DP] = m[r];
            om[w][r][DP + 1] = lt;
        }
    }
    if (W > 1) __syncthreads();
    else __builtin_amdgcn_wave_barrier();
    kv4_finish<T, W, R, DP>(a, wk, om);
}

// 16 query rows of a key/value head: shared heads, several new tokens.  One query row a lane, 16 of the block's 64 tokens
// in each quad of lanes, everything transposed:
//   scores   tokens x queries: lane (quad, n) holds tokens 16 t + 4 quad + 0..3 of query n
//   p s      is an operand as it lies (slots 0-3 from tile 2 ks, 4-7 from 2 ks + 1, the order of the V codes)
//   context  features x queries: lane (quad, n) holds features 16 c + 4 quad + 0..3 of query n
// The (s, z) pairs are one a token and reach the lanes through LDS.
template <typename T, int NG, int W>
__global__ __launch_bounds__(64 * W) void kv4_many_kernel(Kv4AttnArgs a) {
    constexpr bool F32 = sizeof(T) == 4;
    constexpr int QP = F32 ? 3 : 1, PP = F32 ? 3 : 2;
    constexpr int DP = NG * 32;
    __shared__ __align__(16) uint32_t meta[W][2][KV4_TOK * NG];
    __shared__ float om[W][16][DP + 4];

    const int lane = threadIdx.x & 63, w = threadIdx.x >> 6, n = lane & 15, quad = lane >> 4;
    const Kv4Work wk(a, 16);
    bf16x8 qop[QP][NG];
    float qsum[NG];
    const int qi = wk.q0 + n;
    const bool have = qi < a.NQ;
    const int64_t lim = have ? (a.causal ? wk.len - a.Tq + 1 + qi % a.Tq : wk.len) : 0;
    // every row of the block sees at least this many tokens: blocks below it need no comparisons
    const int64_t sure = a.causal ? wk.len - a.Tq + 1 : wk.len;
    {
        const int i = have ? qi % a.Tq : 0, h = wk.hk * a.G + (have ? qi / a.Tq : 0);
        const T* src = (const T*)a.q + wk.b * a.q_bs + h * a.q_hs + i * a.q_ts;
#pragma unroll
        for (int g = 0; g < NG; ++g) {
            const int ch = g * 32 + quad * 8;
            bf16x8 op[QP];
            float sum = kv4_query<T, QP>(src + ch, have && ch < a.dh, op);
            sum += __shfl_xor(sum, 16);
            sum += __shfl_xor(sum, 32);
            qsum[g] = sum * a.scale;
#pragma unroll
            for (int p = 0; p < QP; ++p) qop[p][g] = op[p];
        }
    }
    float m = -INFINITY, l = 0.f, zs[NG];
    f32x4 acc[2 * NG];
#pragma unroll
    for (int g = 0; g < NG; ++g) zs[g] = 0.f;
#pragma unroll
    for (int c = 0; c < 2 * NG; ++c) acc[c] = f32x4{0.f, 0.f, 0.f, 0.f};
    const uint8_t* base = a.data + wk.bh * a.blocks * kv4_block_bytes(NG);
    const float down = KV4_DOWN * a.scale;
    const f32x4 zero4 = {0.f, 0.f, 0.f, 0.f};

    Kv4Tile<NG> cur, nxt;
    if (wk.first + w < wk.last) cur.load(base + (wk.first + w) * kv4_block_bytes(NG), lane);
    for (int64_t blk = wk.first + w; blk < wk.last; blk += W) {
        const bool more = blk + W < wk.last;
        if (more) nxt.load(base + (blk + W) * kv4_block_bytes(NG), lane);
        const bool edge = (blk + 1) * KV4_TOK > sure;
        const int64_t left = lim - blk * KV4_TOK, kept = wk.len - blk * KV4_TOK;
        const int see = (int)(left > KV4_TOK ? KV4_TOK : left);      // tokens of this block that the row sees
#pragma unroll
        for (int g = 0; g < NG; ++g) {
            meta[w][0][lane * NG + g] = lane < kept ? cur.mk[g] : 0u;
            meta[w][1][lane * NG + g] = lane < kept ? cur.mv[g] : 0u;
        }
        __builtin_amdgcn_wave_barrier();
        float s[4][4];
#pragma unroll
        for (int t = 0; t < 4; ++t) {
            f32x4 d[NG];
#pragma unroll
            for (int g = 0; g < NG; ++g) {
                const bf16x8 kop = kv4_k_operand(cur.k[(t * NG + g) >> 2][(t * NG + g) & 3]);
                d[g] = kv4_mfma(kop, qop[0][g], zero4);
#pragma unroll
                for (int p = 1; p < QP; ++p) d[g] = kv4_mfma(kop, qop[p][g], d[g]);
            }
            uint32_t mk[4 * NG];
            __builtin_memcpy(mk, __builtin_assume_aligned(&meta[w][0][(16 * t + 4 * quad) * NG], 16), 16 * NG);
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                float dot = 0.f, off = 0.f;
#pragma unroll
                for (int g = 0; g < NG; ++g) {
                    dot = fmaf(d[g][r], kv4_scale(mk[r * NG + g]), dot);
                    off = fmaf(qsum[g], kv4_zero(mk[r * NG + g]), off);
                }
                s[t][r] = fmaf(dot, down, off);
            }
        }
        if (edge) {
#pragma unroll
            for (int t = 0; t < 4; ++t)
#pragma unroll
                for (int r = 0; r < 4; ++r) s[t][r] = 16 * t + 4 * quad + r < see ? s[t][r] : -INFINITY;
        }
        float top = fmaxf(fmaxf(s[0][0], s[0][1]), fmaxf(s[0][2], s[0][3]));
#pragma unroll
        for (int t = 1; t < 4; ++t) top = fmaxf(top, fmaxf(fmaxf(s[t][0], s[t][1]), fmaxf(s[t][2], s[t][3])));
        if (__any(top - KV4_UPLOG > m + KV4_LAZY)) {
            top = fmaxf(top, __shfl_xor(top, 16));
            top = fmaxf(top, __shfl_xor(top, 32));
            const float mn = fmaxf(m, top - KV4_UPLOG);
            const float f = mn == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(m - mn);
            m = mn;
            l *= f;
#pragma unroll
            for (int g = 0; g < NG; ++g) zs[g] *= f;
#pragma unroll
            for (int c = 0; c < 2 * NG; ++c) acc[c] *= f;
        }
#pragma unroll
        for (int t = 0; t < 4; ++t)
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const bool on = !edge || 16 * t + 4 * quad + r < see;
                s[t][r] = on ? __builtin_amdgcn_exp2f(s[t][r] - m) : 0.f;
                l += s[t][r];
            }
#pragma unroll
        for (int ks = 0; ks < 2; ++ks) {
            uint32_t mv[2][4 * NG];
#pragma unroll
            for (int h = 0; h < 2; ++h)
                __builtin_memcpy(mv[h], __builtin_assume_aligned(&meta[w][1][(32 * ks + 16 * h + 4 * quad) * NG], 16), 16 * NG);
#pragma unroll
            for (int g = 0; g < NG; ++g) {
                bf16x8 pop[PP];
#pragma unroll
                for (int h = 0; h < 2; ++h)
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        const int r = (j >> 1) | ((j & 1) << 1), t = 2 * ks + h;            // order 0 2 1 3
                        const float p = s[t][r];
                        const bool on = !edge || 16 * t + 4 * quad + r < see;
                        float y = p * kv4_scale(mv[h][r * NG + g]);
                        float z = p * kv4_zero(mv[h][r * NG + g]);
                        if (edge) { y = on ? y : 0.f; z = on ? z : 0.f; }
                        zs[g] += z;
#pragma unroll
                        for (int part = 0; part < PP; ++part) {
                            const bf16 b = (bf16)y;
                            y -= (float)b;
                            pop[part][4 * h + j] = b;
                        }
                    }
                const int d = (ks * NG + g) * 2;
                bf16x8 lo, hi;
                kv4_v_operands(cur.v[d >> 2][d & 3], cur.v[d >> 2][(d & 3) + 1], lo, hi);
#pragma unroll
                for (int part = 0; part < PP; ++part) {
                    acc[2 * g] = kv4_mfma(lo, pop[part], acc[2 * g]);
                    acc[2 * g + 1] = kv4_mfma(hi, pop[part], acc[2 * g + 1]);
                }
            }
        }
        __builtin_amdgcn_wave_barrier();
        if (more) cur = nxt;
    }

    l += __shfl_xor(l, 16);
    l += __shfl_xor(l, 32);
#pragma unroll
    for (int g = 0; g < NG; ++g) {
        float z = zs[g];
        z += __shfl_xor(z, 16);
        z += __shfl_xor(z, 32);
        z *= 1.f / KV4_UP;
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
            for (int r = 0; r < 4; ++r)
                om[w][n][g * 32 + h * 16 + quad * 4 + r] = fmaf(acc[2 * g + h][r], h ? KV4_DOWN / 16.f : KV4_DOWN, z);
    }
    if (quad == 0) {
        om[w][n][DP] = m;
        om[w][n][DP + 1] = l * (1.f / KV4_UP);
    }
    if (W > 1) __syncthreads();
    else __builtin_amdgcn_wave_barrier();
    kv4_finish<T, W, 16, DP>(a, wk, om);
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

struct Kv4Shape { int rows, W, splits; int64_t units; };

// How a call is cut: `longest` bounds the lengths (the capacity where the caller knows no better).
static Kv4Shape kv4_shape(int64_t B, int Hkv, int NQ, int64_t longest) {
    Kv4Shape s;
    s.rows = NQ == 1 ? 1 : NQ <= 4 ? 4 : 16;
    s.units = B * Hkv * ((NQ + s.rows - 1) / s.rows);
    const int64_t nb = (longest + KV4_TOK - 1) / KV4_TOK;
    s.W = nb <= 1 || s.units >= 4096 ? 1 : 4;
    const int64_t want = 4096 / (s.units * s.W), most = (nb + s.W - 1) / s.W;
    s.splits = (int)(want < 1 ? 1 : (want > most ? most : want));
    if (s.splits > 512) s.splits = 512;
    return s;
}

template <typename T, int NG, int W>
static void kv4_launch(const Kv4AttnArgs& a, const Kv4Shape& s, hipStream_t st) {
    const unsigned grid = (unsigned)(s.units * s.splits);
    if (s.rows == 1) kv4_few_kernel<T, NG, 1, W><<<grid, 64 * W, 0, st>>>(a);
    else if (s.rows == 4) kv4_few_kernel<T, NG, 4, W><<<grid, 64 * W, 0, st>>>(a);
    else kv4_many_kernel<T, NG, W><<<grid, 64 * W, 0, st>>>(a);
}
template <typename T>
static void kv4_dispatch(const Kv4AttnArgs& a, const Kv4Shape& s, int ng, hipStream_t st) {
#define MSSR_KV4_A(NG)                                \
    case NG:                                          \
        if (s.W == 1) kv4_launch<T, NG, 1>(a, s, st); \
        else kv4_launch<T, NG, 4>(a, s, st);          \
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
    const Kv4Shape s = kv4_shape(c->B, c->H, NQ, kv4_longest(c, longest));
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
    const Kv4Shape s = kv4_shape(c->B, c->H, NQ, kv4_longest(c, longest));
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
