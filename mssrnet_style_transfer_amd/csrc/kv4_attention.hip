// Attention of a few new tokens over a 4-bit key/value cache (layout and numbers: kv4.hpp).
//
// With value = z + s * code per group g of 32 features,
//   q . k_t = sum_g s_tg (sum_{c in g} q_c code_tc) + z_tg (sum_{c in g} q_c)
//   o_c     = (sum_t (p_t s_tg) code_tc + sum_t p_t z_tg) / sum_t p_t
// so the matrix instructions take the CODES as they lie and the scales touch only scores and probabilities: one number
// a token instead of 32.  A code needs no conversion: the bit pattern of an integer c < 1024 read as fp16 is the number
// c * 2^-24 (subnormals, which the matrix cores keep), so `x & 0x000f000f` IS an operand pair and `x & 0x00f000f0` one
// that is 16 times as large.  8 codes take 5 vector instructions.  (The matrix cores align a subnormal's bits as if its
// leading one stood in place: with codes in the lowest four of ten bits, products lose what is below 2^-21 of the largest.
// bf16 scores do not see it; where it counts all codes are 16 times as large, 2^-26, for two shifts more.)
//
// What meets the codes is fp16 too (11 bits), as parts whose products add up in fp32: q one part in bf16 calls (exact), two in
// fp32 ones (2^-22); p s two (2^-22) in either.  One part of p s would keep 2^-12 of the codes' share, which the zeros' share
// nearly cancels: of a single token's stored values, which come back then, one in five was not the nearest bf16 number, and of
// values about zero one in three.  Powers of two keep the parts in fp16's range: a query row is scaled to a largest element in
// [2^13, 2^14) (fp32: [2^9, 2^10); what is 2^-11 of it still has its 22 bits, the rest is off by at most 2^-34 of it).  Every
// query row and group has its own for p s: the largest met so far lies in [2^6, 2^7) when the unit is chosen and may grow to
// 2^15 before it is chosen anew (then the sums shrink); what is 2^-9 of it has its 22 bits, the rest is off by at most 2^-31 of
// it.  With one unit for the largest V scale of all rows, groups and tokens, an fp32 result was 3e-3 off where a value 1e6 times as
// large stood in a token that the row does not attend to.
//
// Where values are spread about zero, codes' and zeros' shares of the context nearly cancel, the more so the more tokens
// there are, and a product's sums are cut, not rounded, where they meet an accumulator that has outgrown them.  7.5 is
// therefore taken from every code (one more product against a constant) and 7.5 s added to every zero, and each block of 64
// tokens starts from zero, added up by rounding additions: fp32 results of 1 .. 16000 tokens of mean zero come out within 1.1e-6
// in norm, and of bf16 ones 1 or 2 in 1000 are not the nearest number.
//
// A wave takes 64 tokens at a time; a row's running maximum moves only when a score passes it by more than 8, and units of
// p s only as above (then that row's sums are rescaled), so that a block of tokens costs one comparison and no cross-lane
// reduction.  The W waves of a block take every W-th 64 tokens of its share of the sentence and are joined through LDS; a second
// launch joins the shares.
#include "kv4.hpp"

namespace mssr {

// Division of a number below 2^31 by one the host knows: a high product, an addition, a shift (Granlund and Montgomery,
// "Division by Invariant Integers using Multiplication", 1994; m = floor(2^32 (2^shift - d) / d) + 1, shift = ceil(log2 d)).
struct Divisor {
    uint32_t d, m, shift;
    Divisor() = default;
    explicit Divisor(uint32_t n) : d(n), shift(0) {
        while (((uint64_t)1 << shift) < n) ++shift;
        m = (uint32_t)((((uint64_t)1 << 32) * (((uint64_t)1 << shift) - n)) / n + 1);
    }
    __device__ __forceinline__ uint32_t operator()(uint32_t x) const { return (__umulhi(m, x) + x) >> shift; }
};

struct Kv4AttnArgs {
    const uint8_t* data;
    int64_t blocks, capacity;
    const void* q;
    void* out;
    int64_t q_bs, q_hs, q_ts, o_bs, o_hs, o_ts;
    Divisor Hkv, Tq;
    int G, dh, causal;              // G query heads share a key/value head
    int NQ;                         // G * Tq query rows of a (sentence, key/value head)
    Divisor splits, chunks;         // chunks of query rows
    IdxTable lengths;
    float scale;                    // of the scores, times log2(e)
    float* part;                    // [rows][splits][dh] unnormalised context, then [rows][splits][2] (max, sum)
    int64_t rows;                   // B * Hkv * NQ
    uint32_t units;                 // pieces of work: B * Hkv * chunks of query rows * splits
};

constexpr float KV4_LAZY = 8.f;          // log2 of how far a probability may pass 1 before a rescale
constexpr int KV4_UP = 7;                // log2 of what the largest p s is held below when its unit is chosen,
constexpr int KV4_FULL = 15;             // and what it may grow to before the unit is chosen anew
constexpr int KV4_MOST_UP = 40;          // no p s is held more than 2^this times: smaller ones are nothing beside the row's sums
constexpr float KV4_NONE = -3e38f;       // the reference of a row that has seen no token: 2^(-inf - KV4_NONE) is 0
constexpr float KV4_MID = 7.5f;          // what is taken from codes and added, times the scale, to zeros
constexpr int KV4_PS_PARTS = 2;          // fp16 parts of p s
constexpr int KV4_MAX_SPLITS = 256;

typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));

// 8 codes of a K dword -> operand whose elements 2 r, 2 r + 1 are features 2 r, 2 r + 1 (r odd, or HIGH: times 16)
template <bool HIGH>
__device__ __forceinline__ f16x8 kv4_k_operand(uint32_t x) {
    constexpr uint32_t lo = 0x000f000fu, hi = 0x00f000f0u;
    const uint32_t y = x >> 8;
    u32x4 r = {HIGH ? (x << 4) & hi : x & lo, x & hi, HIGH ? (x >> 4) & hi : y & lo, y & hi};
    return __builtin_bit_cast(f16x8, r);
}
// two V dwords (4 tokens of tile 2 ks, 4 of tile 2 ks + 1) -> operands of feature n (HIGH: times 16) and of feature 16 + n
// (times 16); the four tokens of a dword come in the order 0 2 1 3
template <bool HIGH>
__device__ __forceinline__ void kv4_v_operands(uint32_t x0, uint32_t x1, f16x8& lo, f16x8& hi) {
    constexpr uint32_t ml = 0x000f000fu, mh = 0x00f000f0u;
    const uint32_t y0 = x0 >> 8, y1 = x1 >> 8;
    u32x4 l = {x0 & ml, y0 & ml, x1 & ml, y1 & ml};
    if (HIGH) l = u32x4{(x0 << 4) & mh, (x0 >> 4) & mh, (x1 << 4) & mh, (x1 >> 4) & mh};
    u32x4 h = {x0 & mh, y0 & mh, x1 & mh, y1 & mh};
    lo = __builtin_bit_cast(f16x8, l);
    hi = __builtin_bit_cast(f16x8, h);
}
// -KV4_MID times 16 in every place
__device__ __forceinline__ f16x8 kv4_mid() {
    constexpr uint32_t w = 0x80788078u;          // -120 * 2^-24, twice
    u32x4 r = {w, w, w, w};
    return __builtin_bit_cast(f16x8, r);
}
__device__ __forceinline__ f32x4 kv4_mfma(f16x8 a, f16x8 b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
}

// Makes a product the fp32 number it is: left alone, the compiler rounds it to fp16 here in one step and there in two, and the
// second part is now and then the rest of another first part.
__device__ __forceinline__ void kv4_pin(float& y) { asm volatile("" : "+v"(y)); }

// Four p s -> half h of their two parts' operands (tokens in the order 0 2 1 3).  bf16 calls cut both parts, two numbers an
// instruction: 2^-20, the same way for all, where the result keeps 2^-8.
template <bool ROUND>
__device__ __forceinline__ void kv4_split(float (&y)[4], f16x8& first, f16x8& second, int h) {
    typedef __fp16 h2 __attribute__((ext_vector_type(2)));
#pragma unroll
    for (int j = 0; j < 2; ++j) {
        float &a = y[j], &b = y[j + 2];
        if (ROUND) {
            kv4_pin(a);
            kv4_pin(b);
            const f16 x = (f16)a, z = (f16)b;
            first[4 * h + 2 * j] = x;
            first[4 * h + 2 * j + 1] = z;
            second[4 * h + 2 * j] = (f16)(a - (float)x);
            second[4 * h + 2 * j + 1] = (f16)(b - (float)z);
        } else {
            const h2 x = __builtin_amdgcn_cvt_pkrtz(a, b);
            const h2 z = __builtin_amdgcn_cvt_pkrtz(a - (float)x[0], b - (float)x[1]);
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                first[4 * h + 2 * j + e] = (f16)x[e];
                second[4 * h + 2 * j + e] = (f16)z[e];
            }
        }
    }
}

// 2^x of a whole number: references of exponents are whole, so that moving one rounds no sum (codes' and zeros' shares of
// the context cancel: rounded apart, an fp32 result of 1000 tokens was off by 1e-5)
__device__ __forceinline__ float kv4_pow2(float x) { return __builtin_amdgcn_ldexpf(1.f, (int)fmaxf(x, -512.f)); }

// What a row holds a group's p s times, as an exponent: as before (but no more than KV4_MOST_UP) where the largest of the
// present ones stays below KV4_FULL, else so that it comes to lie in [2^6, 2^7).  most >= 0; by its bits, for the scalar unit.
__device__ __forceinline__ int kv4_up(int up, float most) {
    const int e = (int)(__builtin_bit_cast(uint32_t, most) >> 23) - 126;         // most < 2^e
    up = up < KV4_MOST_UP ? up : KV4_MOST_UP;
    return e + up > KV4_FULL ? KV4_UP - e : up;
}
// 2^x, x <= 0 (nothing below 2^-126)
__device__ __forceinline__ float kv4_shrink(int x) {
    return __builtin_bit_cast(float, (uint32_t)(x < -127 ? 0 : x + 127) << 23);
}
// the largest of a wave's numbers, none below zero
__device__ __forceinline__ float kv4_wave_most(float v) {
    v = fmaxf(v, dpp_mov<0xB1>(v));
    v = fmaxf(v, dpp_mov<0x4E>(v));
    v = fmaxf(v, dpp_mov<0x141>(v));
    v = fmaxf(v, dpp_mov<0x140>(v));
    v = fmaxf(v, dpp_mov<0x142>(v));             // row_bcast:15, row_bcast:31: the last lane has all
    v = fmaxf(v, dpp_mov<0x143>(v));
    return lane_read(v, 63);
}

// the product of this lane's quad, by two conditions (four nested ones become branches)
__device__ __forceinline__ float kv4_own(float a, float b, float c, float d, bool odd, bool upper) {
    const float lo = odd ? b : a, hi = odd ? d : c;
    return upper ? hi : lo;
}

// A lane's share of a block: 16 NG bytes of K codes, of V codes, and its token's (s, z) pairs.  The next block's K half is
// requested when the scores have used this one's, its V half when the context has: no second set of registers.
template <int NG>
struct Kv4Tile {
    u32x4 k[NG], v[NG];
    uint32_t mk[NG], mv[NG];
    __device__ __forceinline__ void load_k(const uint8_t* blk, int lane, int64_t left = KV4_TOK) {
#pragma unroll
        for (int i = 0; i < NG; ++i)
            if (4 * i / NG < 2 || left > 32) k[i] = *reinterpret_cast<const u32x4*>(blk + i * 1024 + lane * 16);
        __builtin_memcpy(mk, __builtin_assume_aligned(blk + NG * 2048 + lane * (4 * NG), 4), 4 * NG);
    }
    __device__ __forceinline__ void load_v(const uint8_t* blk, int lane, int64_t left = KV4_TOK) {
        __builtin_memcpy(mv, __builtin_assume_aligned(blk + NG * 2304 + lane * (4 * NG), 4), 4 * NG);
#pragma unroll
        for (int i = 0; i < NG; ++i)
            if (2 * i / NG < 1 || left > 32) v[i] = *reinterpret_cast<const u32x4*>(blk + NG * 1024 + i * 1024 + lane * 16);
    }
};

// waves of a block: W work together; of lone ones, four share a block for the sake of the launch (4096 blocks of one wave
// each take longer to start than to run)
constexpr int kv4_waves(int W) { return W == 1 ? 4 : W; }

struct Kv4Work {            // what a block works on: query rows q0 .. of (sentence, key/value head), blocks [first, last)
    int64_t len;
    uint32_t b, bh;
    int hk, q0, split, first, last;     // a sentence has at most 2^30 blocks (the entry point checks it)
    __device__ __forceinline__ Kv4Work(const Kv4AttnArgs& a, int rows, uint32_t id) {
        const uint32_t unit = a.splits(id);
        split = (int)(id - unit * a.splits.d);
        bh = a.chunks(unit);
        q0 = (int)(unit - bh * a.chunks.d) * rows;
        b = a.Hkv(bh);
        hk = (int)(bh - b * a.Hkv.d);
    }
    // query row k of the key/value head: new token i of head h (one row in all: ONE)
    template <bool ONE>
    __device__ __forceinline__ void row(const Kv4AttnArgs& a, int k, int& h, int& i) const {
        const int u = ONE ? 0 : (int)a.Tq((uint32_t)k);
        h = ONE ? hk : hk * a.G + u;
        i = ONE ? 0 : k - u * (int)a.Tq.d;
    }
    __device__ __forceinline__ void span(const Kv4AttnArgs& a) {
        len = a.lengths.at(b);
        len = len < 0 ? 0 : (len > a.capacity ? a.capacity : len);
        const uint32_t nb = (uint32_t)((len + KV4_TOK - 1) >> 6), per = a.splits(nb + a.splits.d - 1);
        const uint32_t lo = (uint32_t)split * per, hi = lo + per;
        first = (int)(lo < nb ? lo : nb);
        last = (int)(hi < nb ? hi : nb);
    }
};

// The features of a query row that this lane multiplies (8 of every group), and the row's scaling.
template <typename T, int NG, int PARTS>
struct Kv4Query {
    f16x8 op[PARTS][NG];        // fp16 parts of q * 2^up; where the code is 16 times as large, a 16th (fp32: everywhere)
    float sum[NG];              // sum of q over the group, every lane of the row
    int up;
    __device__ __forceinline__ void load(const T* src, bool have, int dh, int quad) {
        float x[NG][8], top = 0.f;
#pragma unroll
        for (int g = 0; g < NG; ++g) {
            const int ch = g * 32 + quad * 8;
            const bool in = have && ch < dh;     // the others read the row's first features and drop them
            uint32_t raw[2 * sizeof(T)];
            __builtin_memcpy(raw, src + (in ? ch : 0), sizeof(raw));
#pragma unroll
            for (uint32_t& r : raw) r = in ? r : 0u;
#pragma unroll
            for (int e = 0; e < 8; ++e)
                x[g][e] = __builtin_bit_cast(float, sizeof(T) == 4 ? raw[e % (2 * sizeof(T))]
                                                                   : e & 1 ? raw[e >> 1] & 0xffff0000u : raw[e >> 1] << 16);
#pragma unroll
            for (int e = 0; e < 8; ++e) top = fmaxf(top, fabsf(x[g][e]));
            float t = ((x[g][0] + x[g][1]) + (x[g][2] + x[g][3])) + ((x[g][4] + x[g][5]) + (x[g][6] + x[g][7]));
            t += __shfl_xor(t, 16);
            sum[g] = t + __shfl_xor(t, 32);
        }
        top = fmaxf(top, __shfl_xor(top, 16));
        top = fmaxf(top, __shfl_xor(top, 32));
        up = top > 0.f ? 14 - __builtin_amdgcn_frexp_expf(top) : 0;
#pragma unroll
        for (int g = 0; g < NG; ++g)
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                float y = __builtin_amdgcn_ldexpf(x[g][e], sizeof(T) == 4 || ((e >> 1) & 1) ? up - 4 : up);
#pragma unroll
                for (int p = 0; p < PARTS; ++p) {
                    const f16 h = (f16)y;
                    y -= (float)h;
                    op[p][g][e] = h;
                }
            }
    }
};

// Joins the block's waves (om: per wave and row the context, maximum and sum; synchronised by the caller) and writes the
// row, or its share of it.
template <typename T, int W, int R, int DP>
__device__ __forceinline__ void kv4_finish(const Kv4AttnArgs& a, const Kv4Work& wk, const float (&om)[W][R][DP + 4]) {
    for (int x = W == 1 ? threadIdx.x & 63 : threadIdx.x; x < R * (DP / 2); x += 64 * W) {
        const int r = x / (DP / 2), c = x % (DP / 2) * 2, qi = wk.q0 + r;
        if (qi >= a.NQ || c >= a.dh) continue;
        float top = om[0][r][DP], sum = 0.f, o0 = 0.f, o1 = 0.f;
#pragma unroll
        for (int k = 1; k < W; ++k) top = fmaxf(top, om[k][r][DP]);
#pragma unroll
        for (int k = 0; k < W; ++k) {
            const float mk = om[k][r][DP], lk = om[k][r][DP + 1];
            // a wave that saw nothing has nothing to add (its maximum is minus infinity, like the joint one may be)
            const float f = mk == -INFINITY && lk == 0.f ? 0.f : kv4_pow2(mk - top);
            sum = fmaf(f, lk, sum);
            o0 = fmaf(f, om[k][r][c], o0);
            o1 = fmaf(f, om[k][r][c + 1], o1);
        }
        if (a.splits.d == 1) {
            int h, i;
            wk.template row<R == 1>(a, qi, h, i);
            const float inv = sum == 0.f ? 0.f : 1.f / sum;
            T* dst = (T*)a.out + (int64_t)wk.b * a.o_bs + (int64_t)h * a.o_hs + (int64_t)i * a.o_ts + c;
            dst[0] = from_f<T>(sum == 0.f ? 0.f : o0 * inv);
            dst[1] = from_f<T>(sum == 0.f ? 0.f : o1 * inv);
        } else {
            const int64_t at = ((int64_t)wk.bh * a.NQ + qi) * a.splits.d + wk.split;
            a.part[at * a.dh + c] = o0;
            a.part[at * a.dh + c + 1] = o1;
            if (c == 0) {
                float* ml = a.part + a.rows * a.splits.d * a.dh + at * 2;
                ml[0] = top;
                ml[1] = sum;
            }
        }
    }
}

// Up to 4 query rows (R of them in use) of a key/value head: the decode step.  One token a lane from the scores on.
//   scores   per group 4 products of 16 tokens; every quad of rows of the q operand holds the same rows, so lane
//            (quad, n) finds token n of each product and keeps the one of its own 16 (one fp32 row: its parts are rows)
//   p s      goes through LDS to become an operand: row 4 part + r, the parts add up at the end
// Bound by memory where sentences are long or many: 16 sentences x 8 heads x 26000 tokens of 64 bf16 features (270 MB) 59 us in
// a row of launches over as many caches, 5 of them the join, 4.6 TB/s, the rate of a large copy; 512 x 8 heads x 65 .. 140 tokens
// 13.5 us, 3 of them the launch (35 MB needed, 40 read: half blocks are the least; 12.1 with one part of p s).  By vector
// instructions and latency elsewhere: 8 x 8 heads with 4 fp32 rows each, 4000 .. 8190 tokens of 128 features (63 MB) 29 us, 4 of
// them the join and 10 what a sentence of one block takes as well (some 1800 instructions before and after the loop and 500 for
// the first units; in it 570 vector and 56 matrix ones a block); one sentence of 20 tokens 3.7 us.
template <typename T, int NG, int R, int W>
__global__ __launch_bounds__(64 * kv4_waves(W), 2) void kv4_few_kernel(Kv4AttnArgs a) {
    constexpr bool F32 = sizeof(T) == 4;
    constexpr int PARTS = F32 ? 2 : 1;
    constexpr bool QROWS = F32 && R == 1;        // the parts of q in rows of one product instead of products of their own
    constexpr int PLD = 72;                      // fp16 elements of an LDS row of 64 tokens: 16-byte reads of 16 rows spread
    constexpr int DP = NG * 32;
    __shared__ __align__(16) uint16_t ps_[kv4_waves(W)][NG][KV4_PS_PARTS * R][PLD];
    __shared__ float om_[kv4_waves(W) / W][W][R][DP + 4];

    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), w = W == 1 ? 0 : wave;
    const int lane = threadIdx.x & 63, n = lane & 15, quad = lane >> 4;
    const uint32_t id = W == 1 ? blockIdx.x * 4 + wave : blockIdx.x;
    if (W == 1 && id >= a.units) return;         // (the waves of such a block never wait for each other)
    auto& ps = ps_[wave];
    auto& om = om_[W == 1 ? wave : 0];
    Kv4Work wk(a, R, id);
    const uint8_t* base = a.data + (int64_t)wk.bh * a.blocks * kv4_block_bytes(NG);
    Kv4Tile<NG> cur;
    const bool early = a.splits.d == 1 && w < a.blocks;      // an unsplit wave's first block is known before its length is
    if (early) {
        cur.load_k(base + w * kv4_block_bytes(NG), lane);
        cur.load_v(base + w * kv4_block_bytes(NG), lane);
    }
    wk.span(a);
    f16x8 qop[QROWS ? 1 : PARTS][NG];
    float qsum[R][NG], down[R];                  // scale * sum of q over the group; what a score's codes' part is scaled by
    int64_t lim[R];
    {
        const int r = R == 1 ? 0 : (n & 3), qi = wk.q0 + r;
        const bool have = qi < a.NQ;
        int h, i;
        wk.template row<R == 1>(a, have ? qi : 0, h, i);
        Kv4Query<T, NG, PARTS> q;
        q.load((const T*)a.q + (int64_t)wk.b * a.q_bs + (int64_t)h * a.q_hs + (int64_t)i * a.q_ts, have, a.dh, quad);
        const float back = __builtin_amdgcn_ldexpf(a.scale, 24 - q.up);
#pragma unroll
        for (int rr = 0; rr < R; ++rr) {
            const int k = wk.q0 + rr;
            int hh, ii;
            wk.template row<R == 1>(a, k, hh, ii);
            lim[rr] = k < a.NQ ? (a.causal ? wk.len - (int)a.Tq.d + 1 + ii : wk.len) : 0;
            down[rr] = lane_read(back, rr);
#pragma unroll
            for (int g = 0; g < NG; ++g) qsum[rr][g] = lane_read(q.sum[g] * a.scale, rr);
        }
#pragma unroll
        for (int g = 0; g < NG; ++g) {
            if constexpr (QROWS) {
                const f16x8 none = {};
                qop[0][g] = (n & 3) == 0 ? q.op[0][g] : (n & 3) == 1 ? q.op[PARTS - 1][g] : none;
            } else {
#pragma unroll
                for (int p = 0; p < PARTS; ++p) qop[p][g] = q.op[p][g];
            }
        }
    }

    // m: the running maximum (up to 8 behind), ref: what exponents are taken relative to, ceil(m); l, zs are in units of 2^ref,
    // a group's codes' share in units of 2^(ref - up)
    float m[R], ref[R], l[R], zs[R][NG];
    int up[R][NG];
    bool fresh = true;
    f32x4 acc[2 * NG];
#pragma unroll
    for (int r = 0; r < R; ++r) {
        m[r] = ref[r] = KV4_NONE;
        l[r] = 0.f;
#pragma unroll
        for (int g = 0; g < NG; ++g) {
            zs[r][g] = 0.f;
            up[r][g] = KV4_MOST_UP;
        }
    }
#pragma unroll
    for (int c = 0; c < 2 * NG; ++c) acc[c] = f32x4{0.f, 0.f, 0.f, 0.f};
    // where this lane's token goes among the operand's 64: half, quad, then 0 2 1 3
    const int col = (lane & 32) | ((lane & 12) << 1) | ((lane & 16) >> 2) | ((lane & 1) << 1) | ((lane >> 1) & 1);
    const f32x4 zero4 = {0.f, 0.f, 0.f, 0.f};
    const bool odd = quad & 1, upper = quad & 2;

    const uint8_t* ahead = base + (int64_t)(wk.first + w) * kv4_block_bytes(NG);
    if (!early && wk.first + w < wk.last) {
        cur.load_k(ahead, lane);
        cur.load_v(ahead, lane);
    }
    for (int blk = wk.first + w; blk < wk.last; blk += W) {
        const bool more = blk + W < wk.last;
        ahead += W * kv4_block_bytes(NG);
        const int64_t at = (int64_t)blk * KV4_TOK;
        const bool kept = lane < wk.len - at;
        uint32_t mk[NG], mv[NG];
#pragma unroll
        for (int g = 0; g < NG; ++g) {           // past the sentence's end the cache may hold anything
            mk[g] = kept ? cur.mk[g] : 0u;
            mv[g] = kept ? cur.mv[g] : 0u;
        }
        float dot[R], off[R];
#pragma unroll
        for (int r = 0; r < R; ++r) dot[r] = off[r] = 0.f;
#pragma unroll
        for (int g = 0; g < NG; ++g) {
            f32x4 d[4];
#pragma unroll
            for (int t = 0; t < 4; ++t) {
                const f16x8 kop = kv4_k_operand<F32>(cur.k[(t * NG + g) >> 2][(t * NG + g) & 3]);
                d[t] = kv4_mfma(qop[0][g], kop, zero4);
                if constexpr (PARTS == 2 && !QROWS) d[t] = kv4_mfma(qop[PARTS - 1][g], kop, d[t]);
            }
#pragma unroll
            for (int r = 0; r < R; ++r) {
                float x = kv4_own(d[0][r], d[1][r], d[2][r], d[3][r], odd, upper);
                if constexpr (QROWS) x += kv4_own(d[0][1], d[1][1], d[2][1], d[3][1], odd, upper);
                dot[r] = fmaf(x, kv4_scale(mk[g]), dot[r]);
                off[r] = fmaf(qsum[r][g], kv4_zero(mk[g]), off[r]);
            }
            if (R > 1) __builtin_amdgcn_sched_barrier(0);        // a group at a time, for the registers
        }
        if (more) cur.load_k(ahead, lane, wk.len - at - W * KV4_TOK);
        float s[R];
        uint32_t mask[R];
#pragma unroll
        for (int r = 0; r < R; ++r) {
            const bool see = lane < lim[r] - at;
            s[r] = fmaf(dot[r], down[r], off[r]);
            s[r] = see ? s[r] : -INFINITY;
            // one row sees what the sentence has; of several, each may see less, and a NaN that it does not see is not its
            mask[r] = R == 1 || see ? ~0u : 0u;
        }
        float p[R];
#pragma unroll 1
        for (bool move = fresh;; move = true) {
            if (move) {
                // Every row for itself, so that no row's rounding depends on its neighbours: its reference, then what its groups'
                // p s are held times (as much more as p has become less).
                int rise[R];
#pragma unroll
                for (int r = 0; r < R; ++r) {
                    const float top = wave_max(s[r]);
                    rise[r] = 0;
                    if (top > m[r] + KV4_LAZY) {
                        const float moved = ceilf(top), less = kv4_pow2(ref[r] - moved);
                        rise[r] = __builtin_amdgcn_readfirstlane((int)fminf(moved - ref[r], 512.f));
                        m[r] = lane_read(top, 0);
                        ref[r] = lane_read(moved, 0);
                        l[r] *= less;
#pragma unroll
                        for (int g = 0; g < NG; ++g) zs[r][g] *= less;
                    }
                    p[r] = __builtin_amdgcn_exp2f(s[r] - ref[r]);
                }
#pragma unroll
                for (int g = 0; g < NG; ++g) {
                    f32x4 f = {1.f, 1.f, 1.f, 1.f};
#pragma unroll
                    for (int r = 0; r < R; ++r) {
                        const int next = kv4_up(up[r][g] + rise[r], kv4_wave_most(p[r] * kv4_scale(mv[g] & mask[r])));
                        f[r] = kv4_shrink(next - up[r][g] - rise[r]);
                        up[r][g] = next;
                    }
                    acc[2 * g] *= f;
                    acc[2 * g + 1] *= f;
                }
            }
            bool far = false;
            float big = 0.f;                     // NaN is passed over: it makes its own features NaN and no others
#pragma unroll
            for (int r = 0; r < R; ++r) {
                far |= s[r] > m[r] + KV4_LAZY;
                p[r] = __builtin_amdgcn_exp2f(s[r] - ref[r]);
#pragma unroll
                for (int g = 0; g < NG; ++g) {
                    float y = __builtin_amdgcn_ldexpf(p[r] * kv4_scale(mv[g] & mask[r]), up[r][g]);
                    big = fmaxf(big, y);
#pragma unroll
                    for (int part = 0; part < KV4_PS_PARTS; ++part) {
                        const f16 h = (f16)y;
                        y -= (float)h;
                        ps[g][part * R + r][col] = __builtin_bit_cast(uint16_t, h);
                    }
                }
            }
            asm volatile("" ::: "memory");       // (the parts go to LDS here: kept until after the loop they would be spilled)
            if (move || !__any(far || big > (float)(1 << KV4_FULL))) break;
        }
        fresh = false;
#pragma unroll
        for (int r = 0; r < R; ++r) {
            l[r] += p[r];
#pragma unroll
            for (int g = 0; g < NG; ++g) {
                const uint32_t mvr = mv[g] & mask[r];
                zs[r][g] = fmaf(p[r], fmaf(KV4_MID, kv4_scale(mvr), kv4_zero(mvr)), zs[r][g]);
            }
        }
        __builtin_amdgcn_wave_barrier();
        // rows 4 part + r; the rows past them, and of absent queries, repeat others and are not used
        const int row = R == 1 ? (n >> 2) & 1 : n & 7;
#pragma unroll
        for (int g = 0; g < NG; ++g) {
            f32x4 c0 = zero4, c1 = zero4, mid = zero4;
#pragma unroll
            for (int ks = 0; ks < 2; ++ks) {
                const int d = (ks * NG + g) * 2;
                f16x8 lo, hi;
                kv4_v_operands<true>(cur.v[d >> 2][d & 3], cur.v[d >> 2][(d & 3) + 1], lo, hi);
                const u32x4 raw = *reinterpret_cast<const u32x4*>(&ps[g][row][ks * 32 + quad * 8]);
                const f16x8 pop = __builtin_bit_cast(f16x8, raw);
                c0 = kv4_mfma(pop, lo, c0);
                c1 = kv4_mfma(pop, hi, c1);
                mid = kv4_mfma(pop, kv4_mid(), mid);
            }
            acc[2 * g] += c0 + mid;
            acc[2 * g + 1] += c1 + mid;
        }
        __builtin_amdgcn_wave_barrier();
        if (more) cur.load_v(ahead, lane, wk.len - at - W * KV4_TOK);
    }

#pragma unroll
    for (int r = 0; r < R; ++r) {
        const float lt = wave_sum(l[r]);
        float zt[NG];
#pragma unroll
        for (int g = 0; g < NG; ++g) zt[g] = wave_sum(zs[r][g]);
#pragma unroll
        for (int c = 0; c < 2 * NG; ++c) {
            float u = acc[c][r];
            u += __shfl_xor(u, 16);                             // quads 0 and 1
            u = fmaf(u, __builtin_amdgcn_ldexpf(1.f, 20 - up[r][c >> 1]), zt[c >> 1]);
            if (quad == 0) om[w][r][c * 16 + n] = u;
        }
        if (lane == 0) {
            om[w][r][DP] = m[r] == KV4_NONE ? -INFINITY : ref[r];
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
// Bound by vector instructions (16 scores a lane and block): what can be a product is one, where that rounds nothing that
// cancels.  The zeros' share of a score, sum_g z_tg Q_g, is a product of 8 slots (z exact in fp16, Q in two parts).  The sums of p
// and of p (z + 7.5 s) are fp32 ones of the same p that p s is made of: with p rounded to fp16 in one of them, tokens of equal
// score shared its error, and values about zero came out 2 % (2000 tokens) to 5 % (16000) off.  Scales and zeros are one a
// token and reach the lanes through LDS; a group that is NaN has a NaN scale, its zero is taken as 0 so that rows that do not see
// the token stay clean.
// 24 x 4 heads with 20 rows each, 700 .. 2050 tokens of 96 bf16 features (17 MB): 20.2 us, 7.0 of which a sentence of one block
// takes as well; 15.6 with one part of p s and one unit for all (18.6 then with a second copy of the step for blocks without
// masks and with divisions: code that is run through once is slow to fetch).  104 .. 128 features spill registers (W = 8: 17 in
// bf16 calls, 82 in fp32 ones): the same at 128 features 26 us, in fp32 42.
template <typename T, int NG, int W>
__global__ __launch_bounds__(64 * kv4_waves(W), 2) void kv4_many_kernel(Kv4AttnArgs a) {
    constexpr bool F32 = sizeof(T) == 4;
    constexpr int PARTS = F32 ? 2 : 1;
    constexpr int DP = NG * 32;
    struct Token {
        float vs[NG][KV4_TOK];              // V scales
        uint16_t ks[NG][KV4_TOK];           // K scales
        uint2 kz[KV4_TOK];                  // K zeros, groups 0..3
        float vm[NG][KV4_TOK];              // V zeros and KV4_MID V scales
    };
    __shared__ __align__(16) Token tk[kv4_waves(W)];
    __shared__ float om_[kv4_waves(W) / W][W][16][DP + 4];

    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), w = W == 1 ? 0 : wave;
    const int lane = threadIdx.x & 63, n = lane & 15, quad = lane >> 4;
    const uint32_t id = W == 1 ? blockIdx.x * 4 + wave : blockIdx.x;
    if (W == 1 && id >= a.units) return;
    auto& om = om_[W == 1 ? wave : 0];
    Kv4Work wk(a, 16, id);
    const uint8_t* base = a.data + (int64_t)wk.bh * a.blocks * kv4_block_bytes(NG);
    Kv4Tile<NG> cur;
    const bool early = a.splits.d == 1 && w < a.blocks;
    if (early) {
        cur.load_k(base + w * kv4_block_bytes(NG), lane);
        cur.load_v(base + w * kv4_block_bytes(NG), lane);
    }
    wk.span(a);
    const int qi = wk.q0 + n;
    const bool have = qi < a.NQ;
    int h, i;
    wk.template row<false>(a, have ? qi : 0, h, i);
    const int64_t lim = have ? (a.causal ? wk.len - (int)a.Tq.d + 1 + i : wk.len) : 0;
    // every row of the block sees at least this many tokens: blocks below it need no comparisons (rows that are not there
    // may see anything)
    const int64_t sure = a.causal ? wk.len - (int)a.Tq.d + 1 : wk.len;
    Kv4Query<T, NG, PARTS> q;
    {
        q.load((const T*)a.q + (int64_t)wk.b * a.q_bs + (int64_t)h * a.q_hs + (int64_t)i * a.q_ts, have, a.dh, quad);
    }
    // Q_g * 2^(up - 6) (below 2^13) in two parts: slots 0-3 and 4-7 of quad 0, against z_0..3 twice
    f16x8 qz = {};
    if (quad == 0) {
#pragma unroll
        for (int g = 0; g < NG; ++g) {
            const float y = __builtin_amdgcn_ldexpf(q.sum[g], q.up - 6);
            qz[g] = (f16)y;
            qz[4 + g] = (f16)(y - (float)qz[g]);
        }
    }
    const float down = __builtin_amdgcn_ldexpf(a.scale, 24 - q.up), downz = __builtin_amdgcn_ldexpf(a.scale, 6 - q.up);
    float m = 0.f;                               // (of no meaning while the row is fresh: it has seen no token yet)
    bool fresh = true;
    int up[NG];                                  // p s are held times 2^up, the codes' share with them
    f32x4 acc[2 * NG];
    float zs[NG], l = 0.f;                       // of this lane's tokens
#pragma unroll
    for (int g = 0; g < NG; ++g) {
        zs[g] = 0.f;
        up[g] = KV4_MOST_UP;
    }
#pragma unroll
    for (int c = 0; c < 2 * NG; ++c) acc[c] = f32x4{0.f, 0.f, 0.f, 0.f};
    const f32x4 zero4 = {0.f, 0.f, 0.f, 0.f};
    Token& my = tk[wave];

    auto step = [&](bool edge, int see, const uint32_t (&mv)[NG], const uint8_t* next) {
        float s[4][4];
#pragma unroll
        for (int t = 0; t < 4; ++t) {
            f32x4 d[NG];
#pragma unroll
            for (int g = 0; g < NG; ++g) {
                const f16x8 kop = kv4_k_operand<F32>(cur.k[(t * NG + g) >> 2][(t * NG + g) & 3]);
                d[g] = kv4_mfma(kop, q.op[0][g], zero4);
                if constexpr (PARTS == 2) d[g] = kv4_mfma(kop, q.op[PARTS - 1][g], d[g]);
            }
            const uint2 z2 = my.kz[16 * t + n];
            const u32x4 z4 = {z2.x, z2.y, z2.x, z2.y};
            const f32x4 dz = kv4_mfma(__builtin_bit_cast(f16x8, z4), qz, zero4);
            float dot[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int g = 0; g < NG; ++g) {
                uint32_t k2[2];
                __builtin_memcpy(k2, __builtin_assume_aligned(&my.ks[g][16 * t + 4 * quad], 8), 8);
#pragma unroll
                for (int r = 0; r < 4; ++r) dot[r] = fmaf(d[g][r], kv4_half((k2[r >> 1] >> (16 * (r & 1))) & 0xffffu), dot[r]);
            }
#pragma unroll
            for (int r = 0; r < 4; ++r) s[t][r] = fmaf(dot[r], down, fmaf(dz[r], downz, -m));      // relative to m
            __builtin_amdgcn_sched_barrier(0);   // a tile at a time: all at once would take the registers of a whole wave
        }
        if (next) cur.load_k(next, lane);
        if (edge) {
#pragma unroll
            for (int t = 0; t < 4; ++t)
#pragma unroll
                for (int r = 0; r < 4; ++r) s[t][r] = 16 * t + 4 * quad + r < see ? s[t][r] : -INFINITY;
        }
        float top = fmaxf(fmaxf(s[0][0], s[0][1]), fmaxf(s[0][2], s[0][3]));
#pragma unroll
        for (int t = 1; t < 4; ++t) top = fmaxf(top, fmaxf(fmaxf(s[t][0], s[t][1]), fmaxf(s[t][2], s[t][3])));
        if (__any(top > KV4_LAZY || (fresh && top > -INFINITY))) {
            top = fmaxf(top, __shfl_xor(top, 16));
            top = fmaxf(top, __shfl_xor(top, 32));
            // by how much this row's reference moves: up, or wherever its first tokens are
            const bool moves = fresh ? top > -INFINITY : top > KV4_LAZY;
            const float by = moves ? ceilf(top) : 0.f, less = fresh ? 1.f : kv4_pow2(-by);
            const int rise = fresh ? 0 : (int)fminf(by, 512.f);
            fresh = fresh && !moves;
            m += by;
            l *= less;
#pragma unroll
            for (int g = 0; g < NG; ++g) {
                zs[g] *= less;
                const int next = up[g] + rise < KV4_MOST_UP ? up[g] + rise : KV4_MOST_UP;
                const float f = kv4_shrink(next - up[g] - rise);
                up[g] = next;
                acc[2 * g] *= f;
                acc[2 * g + 1] *= f;
            }
#pragma unroll
            for (int t = 0; t < 4; ++t)
#pragma unroll
                for (int r = 0; r < 4; ++r) s[t][r] -= by;
        }
        bool nan = false;
#pragma unroll
        for (int g = 0; g < NG; ++g) nan |= kv4_scale(mv[g]) != kv4_scale(mv[g]);
        const bool hidden = edge && __any(nan);  // a row may have a NaN scale that it does not see, and 0 times NaN is NaN
#pragma unroll
        for (int g = 0; g < NG; ++g) {
            const float vz = kv4_zero(mv[g]);
            my.vs[g][lane] = kv4_scale(mv[g]);
            my.vm[g][lane] = vz == vz ? fmaf(KV4_MID, kv4_scale(mv[g]), vz) : 0.f;
        }
        __builtin_amdgcn_wave_barrier();
#pragma unroll
        for (int t = 0; t < 4; ++t)
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                s[t][r] = __builtin_amdgcn_exp2f(s[t][r]);
            }
#pragma unroll
        for (int t = 0; t < 4; ++t) l += (s[t][0] + s[t][1]) + (s[t][2] + s[t][3]);
#pragma unroll
        for (int g = 0; g < NG; ++g) {
            // fp32 calls: one accumulator a part, the smaller part's sums would be cut in the larger's (4.7e-6 of 16000 tokens'
            // mean-zero result against 8e-7; bf16 ones have 20 to 40 registers less to spill)
            f32x4 c[PARTS][2], mid = zero4;
#pragma unroll
            for (int part = 0; part < PARTS; ++part) c[part][0] = c[part][1] = zero4;
            float y[4][4], most = 0.f;           // NaN scales are passed over: they make their own features NaN and no others
#pragma unroll
            for (int t = 0; t < 4; ++t) {
                const f32x4 v4 = *reinterpret_cast<const f32x4*>(&my.vs[g][16 * t + 4 * quad]);
                const f32x4 z4 = *reinterpret_cast<const f32x4*>(&my.vm[g][16 * t + 4 * quad]);
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    zs[g] = fmaf(s[t][r], z4[r], zs[g]);
                    y[t][r] = s[t][r] * v4[r];
                }
            }
            if (__builtin_expect(hidden, 0)) {
#pragma unroll
                for (int t = 0; t < 4; ++t)
#pragma unroll
                    for (int r = 0; r < 4; ++r) y[t][r] = 16 * t + 4 * quad + r < see ? y[t][r] : 0.f;
            }
#pragma unroll
            for (int t = 0; t < 4; ++t) most = fmaxf(most, fmaxf(fmaxf(y[t][0], y[t][1]), fmaxf(y[t][2], y[t][3])));
            if (__any(__builtin_amdgcn_ldexpf(most, up[g]) > (float)(1 << KV4_FULL))) {
                most = fmaxf(most, __shfl_xor(most, 16));
                most = fmaxf(most, __shfl_xor(most, 32));
                const int next = kv4_up(up[g], most);
                const float f = kv4_shrink(next - up[g]);
                up[g] = next;
                acc[2 * g] *= f;
                acc[2 * g + 1] *= f;
            }
#pragma unroll
            for (int ks = 0; ks < 2; ++ks) {
                f16x8 pop[KV4_PS_PARTS];
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    float (&part)[4] = y[2 * ks + h];
#pragma unroll
                    for (int r = 0; r < 4; ++r) part[r] = __builtin_amdgcn_ldexpf(part[r], up[g]);
                    kv4_split<F32>(part, pop[0], pop[1], h);
                }
                const int d = (ks * NG + g) * 2;
                f16x8 lo, hi;
                kv4_v_operands<true>(cur.v[d >> 2][d & 3], cur.v[d >> 2][(d & 3) + 1], lo, hi);
#pragma unroll
                for (int part = 0; part < KV4_PS_PARTS; ++part) {
                    c[part % PARTS][0] = kv4_mfma(lo, pop[part], c[part % PARTS][0]);
                    c[part % PARTS][1] = kv4_mfma(hi, pop[part], c[part % PARTS][1]);
                    mid = kv4_mfma(kv4_mid(), pop[part], mid);
                }
                __builtin_amdgcn_sched_barrier(0);
            }
#pragma unroll
            for (int h = 0; h < 2; ++h) acc[2 * g + h] += PARTS == 2 ? c[0][h] + mid + c[PARTS - 1][h] : c[0][h] + mid;
        }
    };

    const uint8_t* ahead = base + (int64_t)(wk.first + w) * kv4_block_bytes(NG);
    if (!early && wk.first + w < wk.last) {
        cur.load_k(ahead, lane);
        cur.load_v(ahead, lane);
    }
    for (int blk = wk.first + w; blk < wk.last; blk += W) {
        const bool more = blk + W < wk.last;
        ahead += W * kv4_block_bytes(NG);
        const int64_t at = (int64_t)blk * KV4_TOK;
        const bool kept = lane < wk.len - at;
        uint32_t z[4] = {0u, 0u, 0u, 0u}, mv[NG];
#pragma unroll
        for (int g = 0; g < NG; ++g) {           // past the sentence's end the cache may hold anything
            const uint32_t mk = kept ? cur.mk[g] : 0u;
            const float kz = kv4_zero(mk);
            mv[g] = kept ? cur.mv[g] : 0u;
            z[g] = kz == kz ? mk >> 16 : 0u;
            my.ks[g][lane] = (uint16_t)mk;
        }
        my.kz[lane] = make_uint2(z[0] | (z[1] << 16), z[2] | (z[3] << 16));
        __builtin_amdgcn_wave_barrier();
        const int64_t left = lim - at;
        step((int64_t)(blk + 1) * KV4_TOK > sure, (int)(left > KV4_TOK ? KV4_TOK : left), mv, more ? ahead : nullptr);
        __builtin_amdgcn_wave_barrier();
        if (more) cur.load_v(ahead, lane);
    }

    l += __shfl_xor(l, 16);
    l += __shfl_xor(l, 32);
#pragma unroll
    for (int g = 0; g < NG; ++g) {
        const float unit = __builtin_amdgcn_ldexpf(1.f, 20 - up[g]);
        float z = zs[g];
        z += __shfl_xor(z, 16);
        z += __shfl_xor(z, 32);
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
            for (int r = 0; r < 4; ++r) om[w][n][g * 32 + h * 16 + quad * 4 + r] = fmaf(acc[2 * g + h][r], unit, z);
    }
    if (quad == 1) {
        om[w][n][DP] = fresh ? -INFINITY : m;
        om[w][n][DP + 1] = l;
    }
    if (W > 1) __syncthreads();
    else __builtin_amdgcn_wave_barrier();
    kv4_finish<T, W, 16, DP>(a, wk, om);
}

// Joins the splits of a query row: the factors once for all, then every wave a quarter of the splits, two features a lane.
// Bound by latency: 4 us of which 3 are a launch's (requesting the first splits before the factors are made changes nothing).
template <typename T>
__global__ __launch_bounds__(256) void kv4_join_kernel(Kv4AttnArgs a) {
    __shared__ float fac[KV4_MAX_SPLITS], red[4][KV4_MAX_DH], sums[4];
    const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
    const int64_t row = blockIdx.x;
    const float2* ml = reinterpret_cast<const float2*>(a.part + a.rows * a.splits.d * a.dh) + row * a.splits.d;
    const float* o = a.part + row * a.splits.d * a.dh;
    float top = -INFINITY;
    for (int s = lane; s < (int)a.splits.d; s += 64) top = fmaxf(top, ml[s].x);      // every wave for itself
    top = wave_max(top);
    float sum = 0.f;
    for (int s = threadIdx.x; s < (int)a.splits.d; s += 256) {
        const float2 x = ml[s];
        const float f = x.x == -INFINITY && x.y == 0.f ? 0.f : kv4_pow2(x.x - top);
        fac[s] = f;
        sum = fmaf(f, x.y, sum);
    }
    sum = wave_sum(sum);
    if (lane == 0) sums[w] = sum;
    __syncthreads();
    sum = (sums[0] + sums[1]) + (sums[2] + sums[3]);
    float o0 = 0.f, o1 = 0.f;
    const int c = 2 * lane;
    if (c < a.dh) {
#pragma unroll 4
        for (int s = w; s < (int)a.splits.d; s += 4) {
            const float2 x = *reinterpret_cast<const float2*>(o + (int64_t)s * a.dh + c);
            o0 = fmaf(fac[s], x.x, o0);
            o1 = fmaf(fac[s], x.y, o1);
        }
        red[w][c] = o0;
        red[w][c + 1] = o1;
    }
    __syncthreads();
    if ((int)threadIdx.x >= a.dh) return;
    const float v = (red[0][threadIdx.x] + red[1][threadIdx.x]) + (red[2][threadIdx.x] + red[3][threadIdx.x]);
    // row = ((b, key/value head), head of its G, new token)
    const uint32_t hi = a.Tq((uint32_t)row), i = (uint32_t)row - hi * a.Tq.d, bh = hi / (uint32_t)a.G, b = a.Hkv(bh);
    const uint32_t h = (bh - b * a.Hkv.d) * a.G + (hi - bh * a.G);
    ((T*)a.out)[b * a.o_bs + h * a.o_hs + i * a.o_ts + threadIdx.x] = from_f<T>(sum == 0.f ? 0.f : v / sum);
}

struct Kv4Shape { int rows, W, splits; int64_t units; };

// How a call is cut: `longest` bounds the lengths (the capacity where the caller knows no better), nb is that in blocks of
// 64 tokens, units the (sentence, key/value head, query rows) triples.  Measured on graph replays, us, "a x b" for a units of b
// tokens, 64 bf16 features unless others are named:
//   a wave each (W = 1) where units fill the chip: 2048 x 140 9.3 against 12.1 with four waves, 4096 x 1200 with 16 rows 110
//     against 127, with 4 rows 79 against 88 (96 fp32 features 134 - 142 against 137); with one row 2048 x 1200 38 against 38
//   eight waves where units are few: 64 x 1200 6.1 against 7.4, 512 x 1200 11.9 against 11.8; but 512 x 300 6.9 against 6.6,
//     512 x 2500 of 128 fp32 features 45 against 41, many-row kernels 512 x 1200 21.2 against 18.5 (256 x 1200 11.5 against 13.9).
//     4 rows: 256 x 2500 16.2 against 18.3, but 64 x 300 7.8 against 7.3
//   splits, whose joining costs a second launch (3 us), where a unit's waves would go round often and the chip has room: as
//     many as give every CU a block, or two where two fit and there are several sentences (their lengths differ), and twice as
//     many again for very long ones.  64 x 10000 15.5 against 26.5 unsplit (with 9 splits, blocks that do not fill the last
//     round, 18.2), 128 fp32 features 25 against 48; 64 x 2500 8.8 against 9.7 unsplit; 128 x 0 .. 32768 30.5 with 8 splits, 31.7
//     with 4, 78 unsplit.  4 rows: 64 x 8190 17 against 30, of 128 fp32 features 28 against 55; 64 x 1000 9.8 against 9.2.  16
//     rows: 64 x 2000 11.3 against 14.4, 64 x 1000 10.2 against 9.4
static Kv4Shape kv4_shape(int64_t B, int Hkv, int NQ, int ng, int64_t longest) {
    Kv4Shape s;
    s.rows = NQ == 1 ? 1 : NQ <= 4 ? 4 : 16;
    s.units = B * Hkv * ((NQ + s.rows - 1) / s.rows);
    const int64_t nb = (longest + KV4_TOK - 1) / KV4_TOK;
    const bool lone = nb <= 1 ? s.rows == 1 || s.units >= 512 : s.units >= 2048 && nb <= (s.rows == 1 ? 16 : 24);
    const bool eight = s.rows == 4    ? nb >= 16 && s.units <= 256
                       : s.units <= 256 ? nb > 4
                                        : s.rows == 1 && ng <= 2 && nb >= 16 && s.units <= 512;
    s.W = lone ? 1 : eight ? 8 : 4;
    int64_t want = 1;
    if (s.rows == 1 && s.units <= 128 && nb * ng >= 80 + s.units / 2)
        want = (s.units < 64 ? 256 : (ng <= 2 ? 512 : 256) << (nb >= 256 ? 1 : 0)) / s.units;
    if (s.rows == 4 && nb * ng >= 48 + s.units / 4) want = 256 / s.units;
    if (s.rows == 16 && nb >= 20) want = 256 / s.units;
    const int64_t most = (nb + s.W - 1) / s.W;
    s.splits = (int)(want < 1 ? 1 : (want > most ? most : want));
    if (s.splits > KV4_MAX_SPLITS) s.splits = KV4_MAX_SPLITS;
    return s;
}

template <typename T, int NG, int W>
static void kv4_launch(const Kv4AttnArgs& a, const Kv4Shape& s, hipStream_t st) {
    const unsigned grid = W == 1 ? (a.units + 3) / 4 : a.units, threads = 64 * kv4_waves(W);
    if (s.rows == 1) kv4_few_kernel<T, NG, 1, W><<<grid, threads, 0, st>>>(a);
    else if (s.rows == 16) kv4_many_kernel<T, NG, W><<<grid, threads, 0, st>>>(a);
    else kv4_few_kernel<T, NG, 4, W><<<grid, threads, 0, st>>>(a);
}
template <typename T>
static void kv4_dispatch(const Kv4AttnArgs& a, const Kv4Shape& s, int ng, hipStream_t st) {
#define MSSR_KV4_A(NG)                                \
    case NG:                                          \
        if (s.W == 1) kv4_launch<T, NG, 1>(a, s, st); \
        else if (s.W == 4) kv4_launch<T, NG, 4>(a, s, st); \
        else kv4_launch<T, NG, 8>(a, s, st);          \
        break;
    switch (ng) { MSSR_KV4_A(1) MSSR_KV4_A(2) MSSR_KV4_A(3) MSSR_KV4_A(4) }
#undef MSSR_KV4_A
    if (a.splits.d > 1) kv4_join_kernel<T><<<(unsigned)a.rows, 256, 0, st>>>(a);
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
    const Kv4Shape s = kv4_shape(c->B, c->H, NQ, kv4_groups(c->dh), kv4_longest(c, longest));
    return s.splits > 1 ? c->B * c->H * NQ * s.splits * (c->dh + 2) * (int64_t)sizeof(float) : 0;
}

extern "C" int mssr_kv4_attention(const mssr_kv4_attention_desc* d, void* stream) {
    MSSR_REQUIRE(d && d->cache, "kv4_attention: null operand");
    const mssr_kv4_cache* c = d->cache;
    const int H = d->H, dtype = d->dtype;
    const int64_t Tq = d->Tq;
    MSSR_REQUIRE(c->data && (Tq == 0 || (d->q && d->out)), "kv4_attention: null operand");
    MSSR_REQUIRE(mssr_kv4_bytes(c->B, c->H, c->capacity, c->dh) > 0 && aligned(c->data, 16),
                 "kv4_attention: cache of %lld x %d heads x %lld tokens x %d features (multiples of 8 up to %d)",
                 (long long)c->B, c->H, (long long)c->capacity, c->dh, KV4_MAX_DH);
    MSSR_REQUIRE(c->capacity <= (int64_t)KV4_TOK << 30, "kv4_attention: %lld tokens a sentence", (long long)c->capacity);
    MSSR_REQUIRE(valid_dtype(dtype), "kv4_attention: dtype %d", dtype);
    MSSR_REQUIRE(Tq >= 0 && H >= c->H && H % c->H == 0, "kv4_attention: %d query heads on %d, %lld rows", H, c->H, (long long)Tq);
    MSSR_REQUIRE(d->lengths || (d->length0 >= 0 && d->length0 <= c->capacity), "kv4_attention: length %lld of a cache of %lld",
                 (long long)d->length0, (long long)c->capacity);
    if (Tq == 0) return MSSR_OK;
    MSSR_REQUIRE(Tq <= (INT32_MAX >> 8) / (H / c->H), "kv4_attention: %lld query rows", (long long)Tq);
    const int NQ = (int)(H / c->H * Tq);
    const Kv4Shape s = kv4_shape(c->B, c->H, NQ, kv4_groups(c->dh), kv4_longest(c, d->longest));
    const int64_t rows = c->B * c->H * NQ;
    MSSR_REQUIRE(s.units <= KV4_MAX_GRID / s.splits && rows <= KV4_MAX_GRID, "kv4_attention: %lld query rows in one call",
                 (long long)rows);
    MSSR_REQUIRE(s.splits == 1 || (d->scratch && d->scratch_bytes >= rows * s.splits * (c->dh + 2) * (int64_t)sizeof(float)),
                 "kv4_attention: scratch of %lld bytes is too small", (long long)d->scratch_bytes);
    Kv4AttnArgs a{(const uint8_t*)c->data, (c->capacity + KV4_TOK - 1) / KV4_TOK, c->capacity, d->q, d->out,
                  d->q_bs, d->q_hs, d->q_ts, d->o_bs, d->o_hs, d->o_ts, Divisor(c->H), Divisor((uint32_t)Tq), H / c->H,
                  c->dh, d->causal ? 1 : 0, NQ, Divisor(s.splits), Divisor((uint32_t)((NQ + s.rows - 1) / s.rows)),
                  {d->lengths, d->lengths_are_64, d->length0}, d->scale * 1.4426950408889634f, (float*)d->scratch, rows,
                  (uint32_t)(s.units * s.splits)};
    if (dtype == MSSR_F32) kv4_dispatch<float>(a, s, kv4_groups(c->dh), (hipStream_t)stream);
    else kv4_dispatch<bf16>(a, s, kv4_groups(c->dh), (hipStream_t)stream);
    MSSR_LAUNCH_OK("kv4_attention");
}
