// kv4.cuh -- the 4-bit K/V cache format shared by its kernels (kv4.cu, kv4_attn.cu, kv4_flash.cu).
//
// A group is the 64 elements of one (token, kv head), stored as 64 nibbles n' + 8 with
// n' in -8..7 and two f16: value = c + d n'.  d has at most 8 significant bits, so d n'
// (|n'| <= 8) is exact in f16 as well as in f32.
// Memory: [slot][kv head][block of 64 tokens], each block 4608 contiguous bytes
//     K codes [64][32] | K (c, d) [64][2] f16 | V codes [64][32] | V (c, d) [64][2] f16
// so a block of keys and values is one bulk copy, and the tokens of one (slot, head)
// are one contiguous stream.  Element i of a group is nibble i % 2 (low first) of byte i / 2.
#pragma once
#include <cuda_fp16.h>
#include <stdint.h>

#include "common.cuh"

namespace madi {

constexpr int kKv4Hd = 64;                              // head_dim
constexpr int kKv4Blk = 64;                             // tokens per block
constexpr int kKv4Codes = kKv4Blk * 32;                 // bytes of one block's K (or V) codes
constexpr int kKv4Half = kKv4Codes + kKv4Blk * 4;       // codes + (c, d)
constexpr int kKv4Block = 2 * kKv4Half;                 // 4608

// 2^e for -126 <= e <= 127.
MADI_DEV float pow2i(int e) { return __uint_as_float((uint32_t)(e + 127) << 23); }
MADI_DEV float max3f(float a, float b, float c) {
    float r;
    asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
    return r;
}

// Keys the query at row i of slot s attends to: rows 0 .. pos[s] + i, or 0 .. lens[s] - 1,
// or the whole cache; never past max_tok.
MADI_DEV int kv4_keys(const uint32_t *pos, const uint32_t *lens, int s, int i, int max_tok) {
    if (pos) {
        const unsigned long long l = (unsigned long long)pos[s] + (unsigned)i + 1u;
        return l < (unsigned long long)max_tok ? (int)l : max_tok;
    }
    if (lens) return lens[s] < (uint32_t)max_tok ? (int)lens[s] : max_tok;
    return max_tok;
}
// Valid rows of slot s among `rows` (the rest is padding).
MADI_DEV int kv4_rows(const uint32_t *n, int s, int rows) {
    return n && n[s] < (uint32_t)rows ? (int)n[s] : rows;
}

}  // namespace madi
