// The 4-bit key/value cache: how it lies in memory, and what the kernels that write, read and attend over it share.
//
// Numbers.  Every group of 32 features of one token and head (the last group of a head may be shorter) is held as
// 4-bit codes with an fp16 scale s and an fp16 zero z:
//   x~ = clamp(x, +-65504),  z = fp16(min x~),  s = fp16((max x~ - min x~) * fp32(1/15)),
//   code = clamp(rint((x~ - z) * (1/s)), 0, 15),   value = z + s * code
// (s = 0: all codes 0; a group that holds a NaN or an infinity has s = z = NaN and reads back as NaN).  5 bits a feature.
//
// Layout.  A (sentence, head) owns ceil(capacity / 64) consecutive blocks of 64 tokens; a block of NG = ceil(dh/32)
// groups is NG * 2560 bytes: K codes (NG * 1024), V codes (NG * 1024), K (s, z) pairs [token][group], V (s, z) pairs.
// The codes lie in the order in which the attention's matrix instructions take them, so that a lane's share is whole
// 16-byte loads and 8 codes become an 8-element operand with one shift and four ANDs (see kv4_attention.hip):
//   K: lane (quad, n) holds, for token 16 t + n and group g, features 32 g + 8 quad + 0..7 in dword t * NG + g;
//      feature 2 r sits in nibble r, feature 2 r + 1 in nibble r + 4
//   V: lane (quad, n) holds, for tokens 32 ks + 16 h + 4 quad + 0..3 (one byte each) of dword (ks * NG + g) * 2 + h,
//      feature 32 g + n in the low and feature 32 g + 16 + n in the high nibble
// and dword d of lane l is at (d / 4) * 1024 + l * 16 + (d % 4) * 4.  A token owns whole bytes in both, so tokens are
// written without reading their neighbours.
#pragma once
#include "common.hpp"

namespace mssr {

constexpr int KV4_TOK = 64;                       // tokens of a block
constexpr int KV4_MAX_DH = 128;
constexpr int64_t KV4_MAX_GRID = (1 << 24) - 1;  // blocks of 256 threads: a grid has fewer than 2^32 threads

typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef _Float16 f16;

constexpr int kv4_groups(int dh) { return (dh + 31) / 32; }
constexpr int64_t kv4_block_bytes(int ng) { return (int64_t)ng * 2560; }

// an index table in 32- or 64-bit integers (null: the same value for every sentence)
struct IdxTable {
    const void* p;
    int is64;
    int64_t uniform;
    __device__ __forceinline__ int64_t at(int64_t i) const {
        if (!p) return uniform;
        return is64 ? reinterpret_cast<const int64_t*>(p)[i] : (int64_t)reinterpret_cast<const int32_t*>(p)[i];
    }
};

__device__ __forceinline__ int kv4_k_off(int ng, int tok, int g, int quad) {
    const int d = (tok >> 4) * ng + g;
    return (d >> 2) * 1024 + (quad * 16 + (tok & 15)) * 16 + (d & 3) * 4;
}
// byte of (token, group g, n); n + 1 is 16 bytes further
__device__ __forceinline__ int kv4_v_off(int ng, int tok, int g, int n) {
    const int d = ((tok >> 5) * ng + g) * 2 + ((tok >> 4) & 1);
    return ng * 1024 + (d >> 2) * 1024 + (((tok >> 2) & 3) * 16 + n) * 16 + (d & 3) * 4 + (tok & 3);
}
__device__ __forceinline__ int kv4_kmeta_off(int ng, int tok, int g) { return ng * 2048 + (tok * ng + g) * 4; }
__device__ __forceinline__ int kv4_vmeta_off(int ng, int tok, int g) { return ng * 2304 + (tok * ng + g) * 4; }

__device__ __forceinline__ float kv4_half(uint32_t bits16) {
    return (float)__builtin_bit_cast(f16, (uint16_t)bits16);
}
__device__ __forceinline__ float kv4_scale(uint32_t meta) { return kv4_half(meta & 0xffffu); }
__device__ __forceinline__ float kv4_zero(uint32_t meta) { return kv4_half(meta >> 16); }

}  // namespace mssr
