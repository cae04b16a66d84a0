// How keys and values lie in a cache of 8-bit codes, and what a code stands for (rotary.hip turns what goes in, kvcache.hip
// writes and reads it, kv_attention.hip attends over it).
//
// A block holds `block` tokens of every head; the codes of one (block, head) are block * D contiguous bytes, in groups of 64
// tokens (64 * D bytes), each in the order in which a wave feeds v_mfma_f32_16x16x32_bf16 from 16-byte loads, so that the 64
// lanes of a load cover 1024 contiguous bytes and nothing has to be transposed on the way to the matrix cores:
//   keys:    [tile of 16 tokens][slab of 16 features][token of the tile][feature of the slab]
//            lane (r = lane & 15, g = lane >> 4) loads slab 4c + g of token r: a row of the operand whose 32 reduced features
//            are 8 of each of the four slabs.
//   values:  [slab of 16 features][g = 0..3][feature][tile t = 0..3][j = 0..3], token = 16 t + 4 g + j
//            lane (n, g) loads, for feature n, the 16 tokens whose probabilities the score product left in that lane's registers.
//
// A code c of a (block, head) stands for c * scale, scale a power of two held in fp32: 1 / scale is a power of two as well, so
// quantising, reading back and moving a block to a larger scale round in one place each, and all of it is exact in bf16.
#pragma once
#include "common.h"

namespace vamd {

typedef __attribute__((ext_vector_type(2))) __bf16 kv_bf16x2;
typedef __attribute__((ext_vector_type(8))) __bf16 kv_bf16x8;
typedef __attribute__((ext_vector_type(2))) float kv_f32x2;
typedef __attribute__((ext_vector_type(4))) float kv_f32x4;
typedef __attribute__((ext_vector_type(16))) float kv_f32x16;
typedef __attribute__((ext_vector_type(2))) uint32_t kv_u32x2;
typedef __attribute__((ext_vector_type(4))) uint32_t kv_u32x4;

constexpr int kKvGroup = 64;                  // tokens of a group
constexpr int kKvListed = 4;                  // see kv_io_units
constexpr int kKvMinExp = -110, kKvMaxExp = 122;

// byte of (token 0..63 of the group, feature d) for D features
__host__ __device__ __forceinline__ int kv_key_at(int token, int d, int D) {
    return (((token >> 4) * (D >> 4) + (d >> 4)) * 16 + (token & 15)) * 16 + (d & 15);
}
__host__ __device__ __forceinline__ int kv_value_at(int token, int d) {
    return (((d >> 4) * 4 + ((token >> 2) & 3)) * 16 + (d & 15)) * 16 + (token >> 4) * 4 + (token & 3);
}

// The other way round: what 16-byte piece q of a group holds.  Keys (S = D / 16 slabs): 16 features from d on of token t; values: of feature d,
// tokens 16 tile + 4 g + 0 .. 3 of the four tiles.
__host__ __device__ __forceinline__ void kv_key_piece(int q, int S, int& t, int& d) {
    t = (q >> 4) / S * 16 + (q & 15);
    d = (q >> 4) % S * 16;
}
__host__ __device__ __forceinline__ void kv_value_piece(int q, int& g, int& d) {
    g = (q >> 4) & 3;
    d = (q >> 6) * 16 + (q & 15);
}

// Four codes (a dword) as floats, and back.  Codes of finite blocks never exceed the largest code: no saturation is needed.
template <int FMT> __device__ __forceinline__ kv_f32x4 kv_decode4(uint32_t w) {
    if (FMT == VAMD_KV_E4M3) {
        const kv_f32x2 a = __builtin_amdgcn_cvt_pk_f32_fp8((int)w, false), b = __builtin_amdgcn_cvt_pk_f32_fp8((int)w, true);
        return kv_f32x4{a[0], a[1], b[0], b[1]};
    }
    return kv_f32x4{(float)(int8_t)w, (float)(int8_t)(w >> 8), (float)(int8_t)(w >> 16), (float)(int8_t)(w >> 24)};
}
template <int FMT> __device__ __forceinline__ uint32_t kv_encode4(float a, float b, float c, float d) {
    if (FMT == VAMD_KV_E4M3) {                          // round to nearest, ties to even
        int w = __builtin_amdgcn_cvt_pk_fp8_f32(a, b, 0, false);
        return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(c, d, w, true);
    }
    const uint32_t x = (uint32_t)(int)rintf(a) & 255u, y = (uint32_t)(int)rintf(b) & 255u;
    const uint32_t z = (uint32_t)(int)rintf(c) & 255u, w = (uint32_t)(int)rintf(d) & 255u;
    return x | y << 8 | z << 16 | w << 24;
}
// Eight codes (two dwords) as the bf16 operand of an MFMA: every code is a bf16 number, nothing is rounded.
template <int FMT> __device__ __forceinline__ kv_bf16x8 kv_operand8(uint32_t lo, uint32_t hi) {
    if (FMT == VAMD_KV_E4M3) {
        const kv_bf16x2 a = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, 1.f, false), b = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, 1.f, true);
        const kv_bf16x2 c = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, 1.f, false), d = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, 1.f, true);
        return kv_bf16x8{a[0], a[1], b[0], b[1], c[0], c[1], d[0], d[1]};
    }
    const kv_f32x4 a = kv_decode4<FMT>(lo), b = kv_decode4<FMT>(hi);
    return kv_bf16x8{(bf16_t)a[0], (bf16_t)a[1], (bf16_t)a[2], (bf16_t)a[3], (bf16_t)b[0], (bf16_t)b[1], (bf16_t)b[2], (bf16_t)b[3]};
}

// Bits of the smallest scale 2^e under which a block whose largest magnitude has the bits `top` needs no code beyond the
// largest one (448 = 1.75 * 2^8; 127 = 1.984375 * 2^6): a comparison of mantissas, no division.  A block that holds an
// infinity or a NaN gets the scale NaN and reads as NaN throughout.  Scales compare as their bits do, NaN above all.
template <int FMT> __host__ __device__ __forceinline__ uint32_t kv_scale_bits(uint32_t top) {
    if (top >= 0x7f800000u) return 0x7fc00000u;
    const int E = (int)(top >> 23) - 127;
    const uint32_t m = top & 0x7fffffu;
    int e = FMT == VAMD_KV_E4M3 ? E - 8 + (m > 0x600000u) : E - 6 + (m > 0x7e0000u);
    e = e < kKvMinExp ? kKvMinExp : e > kKvMaxExp ? kKvMaxExp : e;
    return (uint32_t)(e + 127) << 23;
}

// ---- where a call's rows and blocks are; nothing that a table, a start or an offset holds leads outside the tensors.
// (host code too: tests run these on the CPU)

// Rows of sequence b in a packed batch of `rows`: first .. first + count - 1, of `all` that the sequence has (the others lie beyond
// `most` and are left out).  offsets == NULL: every sequence has `most` rows.
struct KvRows {
    int64_t first;
    int count;
    int64_t all;
};
__host__ __device__ __forceinline__ KvRows kv_rows(const int32_t* offsets, int b, int64_t rows, int most) {
    if (!offsets) return KvRows{(int64_t)b * most, most, most};
    int64_t lo = offsets[b], hi = offsets[b + 1];
    lo = lo < 0 ? 0 : lo > rows ? rows : lo;
    hi = hi < lo ? lo : hi > rows ? rows : hi;
    return KvRows{lo, (int)(hi - lo < most ? hi - lo : most), hi - lo};
}
// Tokens lo .. hi - 1 of the unit (block or group) that starts at position `base`, for rows at start .. start + count - 1.
struct KvSpan {
    int lo, hi;
};
__host__ __device__ __forceinline__ KvSpan kv_span(int64_t start, int count, int64_t base, int unit) {
    if (start < 0) return KvSpan{0, 0};
    const int64_t lo = start > base ? start - base : 0, end = start + count - base;
    const int hi = end < 0 ? 0 : end < unit ? (int)end : unit;
    return KvSpan{lo < unit ? (int)lo : unit, hi};
}
// Units (blocks or groups) that rows at start .. start + count - 1 reach into.
__host__ __device__ __forceinline__ int kv_units(int64_t start, int count, int unit) {
    return start < 0 || count <= 0 ? 0 : (int)((start + count - 1) / unit - start / unit + 1);
}
// How the units of a packed batch are numbered.  By `touched`, which `most` rows reach at worst: unit number / touched of a sequence's, no
// search, but numbers that short sequences lack.  Or (listed) one sequence's units after the other's, as kv_whose finds them: the
// packed rows bound their number, whatever `most` says.  The search costs each workgroup a pass over the sequences before its own, empty
// workgroups cost their launch; written and read back by `touched` / listed (8 heads of 128 features, us): 256 prompts up to 256,
// known to be 67 + 34 / 92 + 45, unknown 1866 + 1340 / 92 + 45; 1000 up to 64, known 161 + 59 / 427 + 188, unknown 7073 + 5075 / 427 + 188; 255 tokens beside a
// prompt of 4000 270 + 182 / 49 + 22 (28 numbers by `touched` for each listed one); 8 prompts up to 4096, known, 33 + 21 / 32 + 20.
struct KvUnits {
    int touched;
    bool listed;
    int64_t count;               // unit numbers a launch has to cover
};
__host__ __device__ __forceinline__ KvUnits kv_io_units(bool packed, int64_t sequences, int64_t rows, int most, int unit) {
    const int touched = (int)(((int64_t)most + unit - 2) / unit + 1);
    const int64_t each = sequences * touched, listed = rows / unit + 2 * sequences;
    return packed && each > kKvListed * listed ? KvUnits{touched, true, listed} : KvUnits{touched, false, each};
}
// Whose is unit `number` among those that the sequences have, units_of(b) of them each, one sequence after the other?  Gives the
// sequence and the unit's number in it, or false behind the last one.  64 sequences at a time, by the whole wave.
template <typename F> __device__ __forceinline__ bool kv_whose(int sequences, int lane, F units_of, uint32_t& number, int& b) {
    for (int b0 = 0; b0 < sequences; b0 += 64) {
        const uint32_t n = b0 + lane < sequences ? (uint32_t)units_of(b0 + lane) : 0u;
        uint32_t upto = n;                                   // (64 of up to 2^25 + 1: within 32 bits)
#pragma unroll
        for (int o = 1; o < 64; o <<= 1) {
            const uint32_t t = __shfl_up(upto, o, 64);
            upto += lane >= o ? t : 0;
        }
        const uint64_t behind = __ballot(upto > number);
        if (behind) {
            const int l = __ffsll((unsigned long long)behind) - 1;
            b = __builtin_amdgcn_readfirstlane(b0 + l);
            number = (uint32_t)__builtin_amdgcn_readfirstlane((int)(number - __shfl(upto - n, l, 64)));
            return true;
        }
        number -= __shfl(upto, 63, 64);
    }
    return false;
}
// The cache's block behind block `blk` of sequence b, or -1: behind the table's end, or a hole.
__host__ __device__ __forceinline__ int kv_page(const int32_t* table, int64_t stride, int width, int blocks, int b, int64_t blk) {
    if (blk < 0 || blk >= width) return -1;
    const int page = table[b * stride + blk];
    return page < 0 || page >= blocks ? -1 : page;
}

}  // namespace vamd
