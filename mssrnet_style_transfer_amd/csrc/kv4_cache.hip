// Writing tokens into the 4-bit key/value cache (layout and numbers: kv4.hpp) and reading them back.
//
// Both directions are bound by memory: a bf16 head of 64 features is 2 * 128 bytes a token on the wide side and 80 on
// the 4-bit side.  Four adjacent lanes share a group of 32 features (8 each: one 16-byte load in bf16); the group's
// minimum and maximum take two quad_perm exchanges.
#include "kv4.hpp"

namespace mssr {

struct Kv4View {
    uint8_t* data;
    int64_t blocks;         // blocks of a (sentence, head)
    int64_t capacity;
    int H, dh;
};

// 8 consecutive features as floats; the address has the element's own alignment only (heads may start anywhere)
template <typename T> struct Ld8;
template <> struct Ld8<float> {
    static __device__ __forceinline__ void load(const float* p, float (&o)[8]) { __builtin_memcpy(o, p, 32); }
    static __device__ __forceinline__ void store(float* p, const float (&o)[8]) { __builtin_memcpy(p, o, 32); }
};
template <> struct Ld8<bf16> {
    static __device__ __forceinline__ void load(const bf16* p, float (&o)[8]) {
        bf16x8 v;
        __builtin_memcpy(&v, p, 16);
#pragma unroll
        for (int i = 0; i < 8; ++i) o[i] = (float)v[i];
    }
    static __device__ __forceinline__ void store(bf16* p, const float (&o)[8]) {
        bf16x8 v;
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = (bf16)o[i];
        __builtin_memcpy(p, &v, 16);
    }
};

template <int CTRL>
__device__ __forceinline__ uint32_t dpp_u32(uint32_t v) {
    return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, CTRL, 0xf, 0xf, true);
}

// The group's codes of this lane's 8 features (one byte each, features 0-3 in c0, 4-7 in c1) and its (s, z) word.
// `live`: the lane holds features (a head's last group may have fewer than 32).  All four lanes of a group call it.
// Bound by vector instructions as soon as memory is not waited for, hence: minima and maxima three at a time, NaN two at a
// time, infinities by the extremes, the elements' clamp by their codes' (x - z, its product with 1/s and its rounding keep order:
// what lies below -65504 has code 0 as -65504 has, what lies above 65504 at most the code of 65504), conversion and packing in
// one instruction.
__device__ __forceinline__ void kv4_quantise(const float (&x)[8], bool live, uint32_t& c0, uint32_t& c1, uint32_t& meta) {
#pragma clang fp contract(off)
    float lo = fminf(fminf(fminf(fminf(x[0], x[1]), x[2]), fminf(fminf(x[3], x[4]), x[5])), fminf(x[6], x[7]));
    float hi = fmaxf(fmaxf(fmaxf(fmaxf(x[0], x[1]), x[2]), fmaxf(fmaxf(x[3], x[4]), x[5])), fmaxf(x[6], x[7]));
    bool nan = __builtin_isunordered(x[0], x[1]) | __builtin_isunordered(x[2], x[3]) | __builtin_isunordered(x[4], x[5]) |
               __builtin_isunordered(x[6], x[7]);
    lo = live ? (nan ? -INFINITY : lo) : INFINITY;
    hi = live ? hi : -INFINITY;
    lo = fminf(lo, dpp_mov<0xB1>(lo));
    hi = fmaxf(hi, dpp_mov<0xB1>(hi));
    lo = fminf(lo, dpp_mov<0x4E>(lo));
    hi = fmaxf(hi, dpp_mov<0x4E>(hi));
    const bool bad = lo == -INFINITY || hi == INFINITY;
    lo = fmaxf(lo, -65504.f);
    hi = fminf(hi, 65504.f);
    lo = fminf(lo, 65504.f);
    hi = fmaxf(hi, -65504.f);
    float step = (hi - lo) * (1.0f / 15.0f);
    // The definition rounds this product to fp32, then to fp16.  Left alone, the compiler takes both in one mixed-precision
    // instruction with a single rounding: another scale in one of some 8000 groups.
    asm volatile("" : "+v"(step));
    const f16 s = (f16)step;
    const f16 z = (f16)lo;
    const float sf = (float)s, zf = (float)z;
    // 1 / s, correctly rounded: one Newton step from the hardware's estimate, checked for every positive fp16 number
    const float r0 = __builtin_amdgcn_rcpf(sf);
    const float inv = sf > 0.f ? __builtin_fmaf(__builtin_fmaf(-sf, r0, 1.f), r0, r0) : 0.f;
    const float most = fminf((65504.f - zf) * inv, 15.f);
    c0 = c1 = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const float q = __builtin_rintf(__builtin_amdgcn_fmed3f((x[i] - zf) * inv, 0.f, most));
        if (i < 4) c0 = __builtin_amdgcn_cvt_pk_u8_f32(q, i, c0);
        else c1 = __builtin_amdgcn_cvt_pk_u8_f32(q, i - 4, c1);
    }
    if (!live || bad) c0 = c1 = 0;
    meta = bad ? 0x7e007e00u
               : (uint32_t)__builtin_bit_cast(uint16_t, s) | ((uint32_t)__builtin_bit_cast(uint16_t, z) << 16);
}

// K dword of the lane: feature 2 r in nibble r, feature 2 r + 1 in nibble r + 4
__device__ __forceinline__ uint32_t kv4_pack_k(uint32_t c0, uint32_t c1) {
    const uint32_t t0 = c0 | (c0 >> 12), t1 = c1 | (c1 >> 12);       // bytes 0, 1: features (0, 2), (1, 3); (4, 6), (5, 7)
    return __builtin_amdgcn_perm(t1, t0, 0x05010400u);
}

// This lane's four V bytes (n0 .. n0 + 3): the low nibbles come from the group's lanes 0 / 1, the high ones from 2 / 3.
__device__ __forceinline__ uint32_t kv4_pack_v(uint32_t c0, uint32_t c1, int quad, int& n0) {
    const uint32_t p0 = dpp_u32<0x4E>(c0), p1 = dpp_u32<0x4E>(c1);       // the lane two further: quad ^ 2
    n0 = (quad & 1) * 8 + (quad >> 1) * 4;
    return quad < 2 ? (c0 | (p0 << 4)) : (p1 | (c1 << 4));
}

struct Kv4WriteArgs {
    Kv4View c;
    const void *k, *v;
    int64_t k_bs, k_hs, k_ts, v_bs, v_hs, v_ts;
    int64_t T;
    IdxTable start, counts;      // counts.p null: all T
    int64_t items;
};

// One group of one token: load, quantise, store straight to memory: a token's bytes are scattered over its block, which costs
// little while there are few.  Bound by latency (512 sentences x 8 heads of 64 bf16 features, one token each: 4.3 us, 2.5 of
// it an empty launch).
template <typename T>
__global__ __launch_bounds__(256) void kv4_write_tokens_kernel(Kv4WriteArgs a) {
    const int64_t id = (int64_t)blockIdx.x * 256 + threadIdx.x;
    const bool on = id < a.items;
    const int ng = kv4_groups(a.c.dh);
    const uint32_t u = on ? (uint32_t)id : 0u;
    const int quad = u & 3;
    const uint32_t w = u >> 2;
    const int g = w % ng;
    const uint32_t row = w / ng;                       // (b, t, h), heads innermost: [B, T, H, dh] memory is read in order
    const int h = row % a.c.H;
    const uint32_t bt = row / a.c.H;
    const int t = bt % (uint32_t)a.T;
    const int64_t b = bt / (uint32_t)a.T;
    const int64_t pos = a.start.at(b) + t;
    const bool keep = on && pos >= 0 && pos < a.c.capacity && (!a.counts.p || t < a.counts.at(b));
    const int ch = g * 32 + quad * 8;
    const bool live = ch < a.c.dh;
    float xk[8] = {}, xv[8] = {};
    if (keep && live) {
        Ld8<T>::load((const T*)a.k + b * a.k_bs + h * a.k_hs + t * a.k_ts + ch, xk);
        Ld8<T>::load((const T*)a.v + b * a.v_bs + h * a.v_hs + t * a.v_ts + ch, xv);
    }
    uint32_t k0, k1, km, v0, v1, vm;
    kv4_quantise(xk, live, k0, k1, km);
    kv4_quantise(xv, live, v0, v1, vm);
    int n0;
    const uint32_t vb = kv4_pack_v(v0, v1, quad, n0);
    if (!keep) return;
    const int tok = pos & (KV4_TOK - 1);
    uint8_t* blk = a.c.data + ((b * a.c.H + h) * a.c.blocks + (pos >> 6)) * kv4_block_bytes(ng);
    *reinterpret_cast<uint32_t*>(blk + kv4_k_off(ng, tok, g, quad)) = kv4_pack_k(k0, k1);
    uint8_t* vp = blk + kv4_v_off(ng, tok, g, n0);
#pragma unroll
    for (int i = 0; i < 4; ++i) vp[16 * i] = (uint8_t)(vb >> (8 * i));
    if (quad == 0) *reinterpret_cast<uint32_t*>(blk + kv4_kmeta_off(ng, tok, g)) = km;
    if (quad == 1) *reinterpret_cast<uint32_t*>(blk + kv4_vmeta_off(ng, tok, g)) = vm;
}

// One cache block of one (sentence, head): its image is put together in LDS and leaves in 16-byte stores where the call
// covers the whole block, in the dwords and bytes of the covered tokens where it does not.  A thread has 8 features of four
// consecutive tokens, so that the V codes, a byte a token, are dwords before they reach LDS.  Bound by memory and, closely, by
// vector instructions: 64 heads x 8191 tokens of 128 bf16 features (268 MB in, 84 out) 92 us, 3.8 TB/s.  (Keys and values
// requested together take 82 us instead of 66 for 8192 heads x 128 tokens: fewer waves fit.)
template <typename T, int NG>
__global__ __launch_bounds__(64 * NG) void kv4_write_blocks_kernel(Kv4WriteArgs a, uint32_t span) {
    constexpr int THREADS = 64 * NG;
    __shared__ __align__(16) uint8_t img[NG * 2560];
    const uint32_t bh = blockIdx.x / span, j = blockIdx.x % span;
    const int64_t b = bh / (uint32_t)a.c.H;
    const int h = bh % (uint32_t)a.c.H;
    const int64_t start = a.start.at(b);
    int64_t cnt = a.counts.p ? a.counts.at(b) : a.T;
    cnt = cnt < 0 ? 0 : (cnt > a.T ? a.T : cnt);
    // tokens [p0, p1) of the cache are written; block j counts from the first one touched
    const int64_t p0 = start < 0 ? 0 : start;
    const int64_t p1 = start > a.c.capacity ? a.c.capacity : (start + cnt > a.c.capacity ? a.c.capacity : start + cnt);
    const int64_t blk = (p0 >> 6) + j, base = blk << 6;
    if (p1 <= p0 || base >= p1) return;
    const int t0 = (int)(p0 > base ? p0 - base : 0), t1 = (int)(p1 - base < KV4_TOK ? p1 - base : KV4_TOK);
    const int quad = threadIdx.x & 3, g = (threadIdx.x >> 2) % NG, tok = (threadIdx.x >> 2) / NG * 4;
    const int ch = g * 32 + quad * 8;
    const bool live = ch < a.c.dh;
#pragma unroll
    for (int which = 0; which < 2; ++which) {
        const int64_t ts = which ? a.v_ts : a.k_ts;
        const T* src = (which ? (const T*)a.v + b * a.v_bs + h * a.v_hs : (const T*)a.k + b * a.k_bs + h * a.k_hs) +
                       (base - start) * ts + ch;
        float x[4][8];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
#pragma unroll
            for (int i = 0; i < 8; ++i) x[e][i] = 0.f;
            if (live && tok + e >= t0 && tok + e < t1) Ld8<T>::load(src + (tok + e) * ts, x[e]);
        }
        uint32_t m[4], vb[4];
        int n0 = 0;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            uint32_t c0, c1;
            kv4_quantise(x[e], live, c0, c1, m[e]);
            if (which) vb[e] = kv4_pack_v(c0, c1, quad, n0);
            else *reinterpret_cast<uint32_t*>(img + kv4_k_off(NG, tok + e, g, quad)) = kv4_pack_k(c0, c1);
        }
        if (which) {                             // four tokens x four bytes, turned over
            const uint32_t a01 = __builtin_amdgcn_perm(vb[1], vb[0], 0x05010400u), b01 = __builtin_amdgcn_perm(vb[1], vb[0], 0x07030602u);
            const uint32_t a23 = __builtin_amdgcn_perm(vb[3], vb[2], 0x05010400u), b23 = __builtin_amdgcn_perm(vb[3], vb[2], 0x07030602u);
            uint32_t* q = reinterpret_cast<uint32_t*>(img + kv4_v_off(NG, tok, g, n0));
            q[0] = __builtin_amdgcn_perm(a23, a01, 0x05040100u);
            q[4] = __builtin_amdgcn_perm(a23, a01, 0x07060302u);
            q[8] = __builtin_amdgcn_perm(b23, b01, 0x05040100u);
            q[12] = __builtin_amdgcn_perm(b23, b01, 0x07060302u);
        }
        // the group's four lanes have the same four pairs; each stores one token's
        const uint32_t lo = quad & 1 ? m[1] : m[0], hi = quad & 1 ? m[3] : m[2];
        *reinterpret_cast<uint32_t*>(img + (which ? kv4_vmeta_off(NG, tok + quad, g) : kv4_kmeta_off(NG, tok + quad, g))) =
            quad & 2 ? hi : lo;
    }
    __syncthreads();
    uint8_t* dst = a.c.data + ((int64_t)bh * a.c.blocks + blk) * kv4_block_bytes(NG);
    if (t0 == 0 && t1 == KV4_TOK) {
        for (int i = threadIdx.x; i < NG * 160; i += THREADS)
            reinterpret_cast<u32x4*>(dst)[i] = reinterpret_cast<const u32x4*>(img)[i];
        return;
    }
    for (int i = threadIdx.x; i < NG * 640; i += THREADS) {
        int lo, n = 1;                                  // tokens [lo, lo + n) of this dword
        if (i < NG * 256) {                             // K codes: one token
            const int d = (i >> 8) * 4 + (i & 3);
            lo = (d / NG) * 16 + ((i >> 2) & 15);
        } else if (i < NG * 512) {                      // V codes: four tokens, a byte each
            const int q = i - NG * 256, d = (q >> 8) * 4 + (q & 3);
            lo = (d / (2 * NG)) * 32 + (d & 1) * 16 + ((q >> 6) & 3) * 4;
            n = 4;
        } else {
            lo = ((i - NG * 512) / NG) & (KV4_TOK - 1); // (s, z) pairs: K's 64 tokens, then V's
        }
        if (lo >= t1 || lo + n <= t0) continue;
        if (lo >= t0 && lo + n <= t1) {
            reinterpret_cast<uint32_t*>(dst)[i] = reinterpret_cast<const uint32_t*>(img)[i];
        } else {
            for (int e = 0; e < 4; ++e)
                if (lo + e >= t0 && lo + e < t1) dst[4 * i + e] = img[4 * i + e];
        }
    }
}

struct Kv4ReadArgs {
    Kv4View c;
    void *k, *v;
    int64_t k_bs, k_hs, k_ts, v_bs, v_hs, v_ts;
    int64_t T;
    IdxTable start, counts;
    int64_t items;
};

// 8 features of K and V of a token from a block's image (memory or LDS)
template <typename P>
__device__ __forceinline__ void kv4_decode(P img, int ng, int tok, int g, int quad, float (&k)[8], float (&v)[8]) {
    const uint32_t kw = *reinterpret_cast<const uint32_t*>(img + kv4_k_off(ng, tok, g, quad));
    const uint32_t km = *reinterpret_cast<const uint32_t*>(img + kv4_kmeta_off(ng, tok, g));
    const uint32_t vm = *reinterpret_cast<const uint32_t*>(img + kv4_vmeta_off(ng, tok, g));
    const float ks = kv4_scale(km), kz = kv4_zero(km), vs = kv4_scale(vm), vz = kv4_zero(vm);
    P vb = img + kv4_v_off(ng, tok, g, (quad & 1) * 8);
    const int sh = (quad >> 1) * 4;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        k[j] = fmaf(ks, (float)((kw >> (4 * ((j >> 1) + 4 * (j & 1)))) & 0xfu), kz);     // s * code is exact: one rounding
        v[j] = fmaf(vs, (float)((vb[16 * j] >> sh) & 0xf), vz);
    }
}

// The same items the other way, 4.2 us for 4096 heads x 1 token.
template <typename T>
__global__ __launch_bounds__(256) void kv4_read_tokens_kernel(Kv4ReadArgs a) {
    const int64_t id = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (id >= a.items) return;
    const int ng = kv4_groups(a.c.dh);
    const uint32_t u = (uint32_t)id;
    const int quad = u & 3;
    const uint32_t w = u >> 2;
    const int g = w % ng;
    const uint32_t row = w / ng;
    const int h = row % a.c.H;
    const uint32_t bt = row / a.c.H;
    const int t = bt % (uint32_t)a.T;
    const int64_t b = bt / (uint32_t)a.T;
    const int ch = g * 32 + quad * 8;
    if (ch >= a.c.dh) return;
    const int64_t pos = a.start.at(b) + t;
    float k[8] = {}, v[8] = {};
    if (pos >= 0 && pos < a.c.capacity && (!a.counts.p || t < a.counts.at(b)))
        kv4_decode((const uint8_t*)a.c.data + ((b * a.c.H + h) * a.c.blocks + (pos >> 6)) * kv4_block_bytes(ng), ng,
                   (int)(pos & (KV4_TOK - 1)), g, quad, k, v);
    Ld8<T>::store((T*)a.k + b * a.k_bs + h * a.k_hs + t * a.k_ts + ch, k);
    Ld8<T>::store((T*)a.v + b * a.v_bs + h * a.v_hs + t * a.v_ts + ch, v);
}

// 64 output tokens of one (sentence, head); they lie in at most two cache blocks, whose images pass through LDS.  Bound by
// memory: 64 heads x 8191 tokens of 128 bf16 features 66 us, 5.3 TB/s.
template <typename T, int NG>
__global__ __launch_bounds__(256) void kv4_read_blocks_kernel(Kv4ReadArgs a, uint32_t span) {
    __shared__ __align__(16) uint8_t img[2 * NG * 2560];
    const uint32_t bh = blockIdx.x / span, j = blockIdx.x % span;
    const int64_t b = bh / a.c.H;
    const int h = bh % a.c.H;
    const int64_t start = a.start.at(b);
    int64_t cnt = a.counts.p ? a.counts.at(b) : a.T;
    const int64_t o0 = (int64_t)j * KV4_TOK;
    const int nt = (int)(a.T - o0 < KV4_TOK ? a.T - o0 : KV4_TOK);
    const int64_t pos0 = start + o0;                    // cache position of the first output token
    const int64_t first = pos0 >> 6;                    // its block (arithmetic shift: a negative start stays below 0)
#pragma unroll
    for (int s = 0; s < 2; ++s) {
        const int64_t blk = first + s;
        if (blk < 0 || blk >= a.c.blocks || (blk << 6) >= pos0 + nt) continue;
        const u32x4* src = reinterpret_cast<const u32x4*>(a.c.data + ((int64_t)bh * a.c.blocks + blk) * kv4_block_bytes(NG));
        u32x4* d = reinterpret_cast<u32x4*>(img + s * NG * 2560);
        for (int i = threadIdx.x; i < NG * 160; i += 256) d[i] = src[i];
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < NG; ++i) {
        const int item = i * 256 + threadIdx.x, quad = item & 3, g = (item >> 2) % NG, tok = (item >> 2) / NG;
        const int ch = g * 32 + quad * 8;
        if (tok >= nt || ch >= a.c.dh) continue;
        const int64_t pos = pos0 + tok;
        float k[8] = {}, v[8] = {};
        if (pos >= 0 && pos < a.c.capacity && o0 + tok < cnt)
            kv4_decode((const uint8_t*)img + (int)((pos >> 6) - first) * NG * 2560, NG, (int)(pos & (KV4_TOK - 1)), g, quad, k, v);
        Ld8<T>::store((T*)a.k + b * a.k_bs + h * a.k_hs + (o0 + tok) * a.k_ts + ch, k);
        Ld8<T>::store((T*)a.v + b * a.v_bs + h * a.v_hs + (o0 + tok) * a.v_ts + ch, v);
    }
}

static int kv4_check(const mssr_kv4_cache* c, const char* who) {
    MSSR_REQUIRE(c && c->data, "%s: no cache", who);
    MSSR_REQUIRE(c->B >= 1 && c->H >= 1 && c->capacity >= 1 && c->dh >= 8 && c->dh <= KV4_MAX_DH && c->dh % 8 == 0,
                 "%s: cache of %lld x %d heads x %lld tokens x %d features (multiples of 8 up to %d)", who, (long long)c->B,
                 c->H, (long long)c->capacity, c->dh, KV4_MAX_DH);
    MSSR_REQUIRE(aligned(c->data, 16), "%s: the cache must be 16-byte aligned", who);
    return MSSR_OK;
}
static int kv4_check_rows(const mssr_kv4_rows* r, const char* who) {
    MSSR_REQUIRE(r, "%s: no descriptor", who);
    if (int rc = kv4_check(r->cache, who)) return rc;
    MSSR_REQUIRE(r->T == 0 || (r->k && r->v), "%s: null keys or values", who);
    MSSR_REQUIRE(valid_dtype(r->dtype), "%s: dtype %d", who, r->dtype);
    MSSR_REQUIRE(r->T >= 0, "%s: %lld tokens", who, (long long)r->T);
    MSSR_REQUIRE((r->index_bits & ~3) == 0, "%s: index_bits %d", who, r->index_bits);
    const int64_t capacity = r->cache->capacity;
    MSSR_REQUIRE(r->start || (r->start0 >= 0 && r->T <= capacity && r->start0 <= capacity - r->T),
                 "%s: %lld tokens from %lld on in a cache of %lld", who, (long long)r->T, (long long)r->start0,
                 (long long)capacity);
    return MSSR_OK;
}
static Kv4View kv4_view(const mssr_kv4_cache* c) {
    return Kv4View{(uint8_t*)c->data, (c->capacity + KV4_TOK - 1) / KV4_TOK, c->capacity, c->H, c->dh};
}

}  // namespace mssr

using namespace mssr;

extern "C" int64_t mssr_kv4_bytes(int64_t B, int H, int64_t capacity, int dh) {
    if (B < 1 || H < 1 || capacity < 1 || dh < 8 || dh > KV4_MAX_DH || dh % 8) return -1;
    if (capacity > (int64_t)1 << 40 || B > ((int64_t)1 << 40) / H) return -1;
    const int64_t per = ((capacity + KV4_TOK - 1) / KV4_TOK) * kv4_block_bytes(kv4_groups(dh));
    if (per > INT64_MAX / (B * H)) return -1;
    return B * H * per;
}

// Whether a call goes token by token (else by blocks, through LDS).  Graph replays, us, tokens against blocks:
//   writing: below 64 tokens a sentence no block is whole (8192 heads of 64 features: 2 tokens 6.1 against 56, 32 tokens 34
//     against 58, 64 tokens 61 against 54, 128 tokens 127 against 66), and a block's work takes 5 us however few there are
//     (64 heads x 192 tokens 4.6 against 6.1, 8 heads x 4000 tokens 7.3 against 7.6, but 256 heads of 128 features x 128
//     tokens 11 against 8.2)
//   reading: the other way round from 16 tokens on (8192 heads: 8 tokens 9.9 against 13, 16 tokens 15.7 against 14.0; 64
//     heads x 16 tokens 2.8 against 2.5)
// and what 32-bit item numbers hold.
static bool kv4_by_tokens(int64_t bh, int64_t T, int ng, bool write) {
    if (bh > (int64_t)1 << 27 || T >= (int64_t)1 << 26) return false;
    const bool few = write ? T < KV4_TOK || bh * T * ng <= 1 << 16 : T < 16;
    return few && bh * T * ng * 4 < (int64_t)1 << 31;
}

extern "C" int mssr_kv4_write(const mssr_kv4_rows* r, void* stream) {
    if (int rc = kv4_check_rows(r, "kv4_write")) return rc;
    const mssr_kv4_cache* c = r->cache;
    const int64_t T = r->T;
    const int dtype = r->dtype;
    if (T == 0) return MSSR_OK;
    const int ng = kv4_groups(c->dh);
    hipStream_t s = (hipStream_t)stream;
    Kv4WriteArgs a{kv4_view(c), r->k, r->v, r->k_bs, r->k_hs, r->k_ts, r->v_bs, r->v_hs, r->v_ts, T,
                  {r->start, r->index_bits & 1, r->start0}, {r->counts, (r->index_bits >> 1) & 1, 0}, 0};
    const int64_t bh = c->B * c->H;
    if (kv4_by_tokens(bh, T, ng, true)) {
        a.items = bh * T * ng * 4;
        const unsigned grid = (unsigned)((a.items + 255) / 256);
        if (dtype == MSSR_F32) kv4_write_tokens_kernel<float><<<grid, 256, 0, s>>>(a);
        else kv4_write_tokens_kernel<bf16><<<grid, 256, 0, s>>>(a);
    } else {
        const int64_t touched = (T + KV4_TOK - 2) / KV4_TOK + 1;    // blocks that T tokens from anywhere can reach
        const int64_t span = touched < a.c.blocks ? touched : a.c.blocks;
        MSSR_REQUIRE(bh <= KV4_MAX_GRID / span, "kv4_write: %lld heads x %lld blocks in one call", (long long)bh, (long long)span);
        const unsigned grid = (unsigned)(bh * span);
#define MSSR_KV4_W(NG)                                                                                   \
    case NG:                                                                                             \
        if (dtype == MSSR_F32) kv4_write_blocks_kernel<float, NG><<<grid, 64 * NG, 0, s>>>(a, (uint32_t)span); \
        else kv4_write_blocks_kernel<bf16, NG><<<grid, 64 * NG, 0, s>>>(a, (uint32_t)span);                  \
        break;
        switch (ng) { MSSR_KV4_W(1) MSSR_KV4_W(2) MSSR_KV4_W(3) MSSR_KV4_W(4) }
#undef MSSR_KV4_W
    }
    MSSR_LAUNCH_OK("kv4_write");
}

extern "C" int mssr_kv4_read(const mssr_kv4_rows* r, void* stream) {
    if (int rc = kv4_check_rows(r, "kv4_read")) return rc;
    const mssr_kv4_cache* c = r->cache;
    const int64_t T = r->T;
    const int dtype = r->dtype;
    if (T == 0) return MSSR_OK;
    const int ng = kv4_groups(c->dh);
    hipStream_t s = (hipStream_t)stream;
    Kv4ReadArgs a{kv4_view(c), r->k, r->v, r->k_bs, r->k_hs, r->k_ts, r->v_bs, r->v_hs, r->v_ts, T,
                  {r->start, r->index_bits & 1, r->start0}, {r->counts, (r->index_bits >> 1) & 1, 0}, 0};
    const int64_t bh = c->B * c->H;
    if (kv4_by_tokens(bh, T, ng, false)) {
        a.items = bh * T * ng * 4;
        const unsigned grid = (unsigned)((a.items + 255) / 256);
        if (dtype == MSSR_F32) kv4_read_tokens_kernel<float><<<grid, 256, 0, s>>>(a);
        else kv4_read_tokens_kernel<bf16><<<grid, 256, 0, s>>>(a);
    } else {
        const int64_t span = (T + KV4_TOK - 1) / KV4_TOK;
        MSSR_REQUIRE(bh <= KV4_MAX_GRID / span, "kv4_read: %lld heads x %lld blocks in one call", (long long)bh, (long long)span);
        const unsigned grid = (unsigned)(bh * span);
#define MSSR_KV4_R(NG)                                                                                   \
    case NG:                                                                                             \
        if (dtype == MSSR_F32) kv4_read_blocks_kernel<float, NG><<<grid, 256, 0, s>>>(a, (uint32_t)span);  \
        else kv4_read_blocks_kernel<bf16, NG><<<grid, 256, 0, s>>>(a, (uint32_t)span);                   \
        break;
        switch (ng) { MSSR_KV4_R(1) MSSR_KV4_R(2) MSSR_KV4_R(3) MSSR_KV4_R(4) }
#undef MSSR_KV4_R
    }
    MSSR_LAUNCH_OK("kv4_read");
}
