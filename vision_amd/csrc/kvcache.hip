// Writing keys and values into a cache of 8-bit codes with one power-of-two scale for each (block of tokens, head), and reading
// them back.  The layout, the codes and the scales are described in kv_layout.h.
//
// One workgroup per (sequence, touched block, keys or values, head).  Writing:
//   1. the largest magnitude of the call's rows in this block, as an integer maximum over bit patterns;
//   2. the scale: for a block that the call begins at its first token, what that maximum needs; otherwise the larger of that and
//      the block's scale.  A scale is a power of two, so moving a block to a larger one is an exact product by old / new in
//      32 bits and one rounding to the code: e4m3 codes only lose bits that fall below the smallest code, int8 codes round again;
//   3. the rows as codes, from registers where a workgroup can hold them, else read again (from L2): x * 2^-e is exact, the code's
//      rounding (to nearest, ties to even) is the only one.
// Bound by memory: 16000 tokens of 8 heads and 128 features (int8, blocks of 128) 29 us written, 21 read back, 3.4 and 4.6
// TB/s.  A block belongs to one sequence while it is written: no two
// workgroups of a call write the same bytes, nothing is added atomically, the result does not depend on any order.
#include "kv_layout.h"

namespace vamd {

struct KvIoArgs {
    const void* x[2];            // append: rows in (keys, values); read: unused
    void* y[2];                  // read: rows out
    int64_t tok[2], head[2];     // strides of those rows, in elements
    uint8_t* codes[2];
    float* scales[2];
    const int32_t* table;        // [sequences][table_stride], `width` entries used
    int64_t table_stride;
    const int32_t* start;        // position of a sequence's first row
    const int32_t* offsets;
    int64_t rows;
    int sequences, heads, D, block, width, blocks, most, touched;
    bool listed;                 // see KvUnits
};

// Unit number `id` of a launch: sequence b's j-th, or false where there is none.
__device__ __forceinline__ bool kv_io_unit(const KvIoArgs& a, int64_t id, int unit, int& j, int& b) {
    if (a.listed) {
        uint32_t number = (uint32_t)id;
        const bool found = kv_whose(a.sequences, (int)(threadIdx.x & 63), [&](int s) {
            return kv_units(a.start[s], kv_rows(a.offsets, s, a.rows, a.most).count, unit);
        }, number, b);
        j = (int)number;
        return found;
    }
    j = (int)(id % a.touched);
    b = (int)(id / a.touched);
    return b < a.sequences;
}

template <typename T, bool ALIGNED> __device__ __forceinline__ Vec16<T> kv_load16(const T* p) {
    if (ALIGNED) return *(const Vec16<T>*)p;
    Vec16<T> w;
#pragma unroll
    for (int e = 0; e < Vec16<T>::N; ++e) w.v[e] = p[e];
    return w;
}
template <typename T, bool ALIGNED> __device__ __forceinline__ void kv_load8(const T* p, float (&v)[8]) {
    if (ALIGNED) {
#pragma unroll
        for (int i = 0; i < 8 / Vec16<T>::N; ++i) {
            const Vec16<T> w = *(const Vec16<T>*)(p + i * Vec16<T>::N);
#pragma unroll
            for (int e = 0; e < Vec16<T>::N; ++e) v[i * Vec16<T>::N + e] = to_f(w.v[e]);
        }
    } else {
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = to_f(p[e]);
    }
}
template <typename T, bool ALIGNED> __device__ __forceinline__ void kv_store8(T* p, const float (&v)[8]) {
    if (ALIGNED) {
#pragma unroll
        for (int i = 0; i < 8 / Vec16<T>::N; ++i) {
            Vec16<T> w;
#pragma unroll
            for (int e = 0; e < Vec16<T>::N; ++e) w.v[e] = from_f<T>(v[i * Vec16<T>::N + e]);
            *(Vec16<T>*)(p + i * Vec16<T>::N) = w;
        }
    } else {
#pragma unroll
        for (int e = 0; e < 8; ++e) p[e] = from_f<T>(v[e]);
    }
}

// Transposes the 4 x 4 dwords of four neighbouring lanes: lane j (0..3) gives r[i] to lane i and gets theirs in order.
__device__ __forceinline__ void kv_transpose_quad(kv_u32x4& r, int j) {
    auto trade = [&](int a, int b, bool upper, auto swap) {
        const uint32_t got = swap(upper ? r[a] : r[b]);
        r[a] = upper ? got : r[a];
        r[b] = upper ? r[b] : got;
    };
    auto by1 = [](uint32_t x) { return (uint32_t)__builtin_amdgcn_mov_dpp((int)x, 0xb1, 0xf, 0xf, true); };      // lanes 1 0 3 2
    auto by2 = [](uint32_t x) { return (uint32_t)__builtin_amdgcn_mov_dpp((int)x, 0x4e, 0xf, 0xf, true); };      // lanes 2 3 0 1
    trade(0, 1, j & 1, by1);
    trade(2, 3, j & 1, by1);
    trade(0, 2, j & 2, by2);
    trade(1, 3, j & 2, by2);
}

template <int FMT> __device__ __forceinline__ uint32_t kv_rescale4(uint32_t w, float ratio) {
    const kv_f32x4 v = kv_decode4<FMT>(w);
    return kv_encode4<FMT>(v[0] * ratio, v[1] * ratio, v[2] * ratio, v[3] * ratio);
}

template <typename T, int FMT, bool ALIGNED, int HOLD>
__global__ void __launch_bounds__(256) kv_append_kernel(const KvIoArgs a) {
    __shared__ uint32_t tops[4];
    int64_t id = block_number();
    const int h = (int)(id % a.heads);
    id /= a.heads;
    const int kv = (int)(id & 1);
    id >>= 1;
    int j, b;
    if (!kv_io_unit(a, id, a.block, j, b)) return;
    const int64_t start = a.start[b];
    const KvRows rows = kv_rows(a.offsets, b, a.rows, a.most);
    const int64_t blk = start / a.block + j, base = blk * a.block;
    const KvSpan span = kv_span(start, rows.count, base, a.block);
    const int lo = span.lo, hi = span.hi;
    if (hi <= lo) return;
    const int page = kv_page(a.table, a.table_stride, a.width, a.blocks, b, blk);
    if (page < 0) return;

    const int tid = threadIdx.x, nt = blockDim.x, D = a.D, P = D >> 3, S = D >> 4;
    const int64_t tok = a.tok[kv];
    const T* x = (const T*)a.x[kv] + (rows.first + base - start) * tok + h * a.head[kv];     // row of token 0 of the block
    // What a lane quantises later it keeps in registers where that is little (HOLD times 32 elements): pieces of keys are 16
    // features of a token, of values 8 features of 4 neighbouring tokens; `pieces` and `quads` of them in a group of 64 tokens.
    const int pieces = kKvGroup * S, quads = 16 * P;
    const int f0 = lo / kKvGroup, f1 = (hi + kKvGroup - 1) / kKvGroup;          // groups with fresh tokens
    const int items = (f1 - f0) * (kv == 0 ? pieces : quads), per = kv == 0 ? 2 * HOLD : HOLD;
    const bool held = items <= per * nt;
    auto key_place = [&](int i, int& g, int& t, int& d) {
        g = i / pieces;
        kv_key_piece(i - g * pieces, S, t, d);
        t += g * kKvGroup;
    };
    auto value_place = [&](int i, int& g, int& t, int& p, int& gg, int& tt) {
        g = i / quads;
        const int q = i - g * quads;
        tt = q & 3;
        p = (q >> 2) % P;
        gg = (q >> 2) / P;
        t = g * kKvGroup + tt * 16 + gg * 4;
    };
    Vec16<T> kept[HOLD][32 * sizeof(T) / 16];
    uint32_t top = 0;
    auto look = [&](const Vec16<T>& w) {
#pragma unroll
        for (int e = 0; e < Vec16<T>::N; ++e) {
            const uint32_t m = __float_as_uint(to_f(w.v[e])) & 0x7fffffffu;
            top = m > top ? m : top;
        }
    };
    constexpr int V8 = 8 / Vec16<T>::N;                          // 16-byte vectors of 8 elements
    if (held && kv == 0) {
#pragma unroll
        for (int n = 0; n < 2 * HOLD; ++n) {
            int g, t = hi, d = 0;
            const int i = tid + n * nt;
            if (i < items) key_place(i + f0 * pieces, g, t, d);
#pragma unroll
            for (int e = 0; e < 2 * V8; ++e) {
                Vec16<T> w = {};
                if (t >= lo && t < hi) w = kv_load16<T, ALIGNED>(x + t * tok + d + e * Vec16<T>::N);
                kept[n >> 1][(n & 1) * 2 * V8 + e] = w;
            }
        }
    } else if (held) {
#pragma unroll
        for (int n = 0; n < HOLD; ++n) {
            int g, t = hi, p = 0, gg, tt;
            const int i = tid + n * nt;
            if (i < items) value_place(i + f0 * quads, g, t, p, gg, tt);
#pragma unroll
            for (int e = 0; e < 4 * V8; ++e) {
                Vec16<T> w = {};
                const int tn = t + e / V8;
                if (tn >= lo && tn < hi) w = kv_load16<T, ALIGNED>(x + tn * tok + p * 8 + e % V8 * Vec16<T>::N);
                kept[n][e] = w;
            }
        }
    }
    if (held) {
#pragma unroll
        for (int n = 0; n < HOLD; ++n)
#pragma unroll
            for (int e = 0; e < 4 * V8; ++e) look(kept[n][e]);
    } else {
        for (int i = tid; i < (hi - lo) * P; i += nt) {
            const int t = lo + i / P, p = i % P;
#pragma unroll
            for (int e = 0; e < V8; ++e) look(kv_load16<T, ALIGNED>(x + t * tok + p * 8 + e * Vec16<T>::N));
        }
    }
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) {
        const uint32_t m = __shfl_xor(top, o, 64);
        top = m > top ? m : top;
    }
    float* scale = a.scales[kv] + (int64_t)page * a.heads + h;
    const uint32_t old = lo > 0 ? __float_as_uint(*scale) : 0u;
    if (nt > 64) {
        if ((tid & 63) == 0) tops[tid >> 6] = top;
        __syncthreads();
#pragma unroll
        for (int w = 0; w < 4; ++w) top = tops[w] > top ? tops[w] : top;
    }
    const uint32_t need = kv_scale_bits<FMT>(top), now = need > old ? need : old;
    const bool dead = now >= 0x7f800000u;                        // the block reads as NaN, whatever its codes
    const float inv = dead ? 0.f : __uint_as_float(0x7f000000u - now);          // 2^-e
    // under the largest scale the upper codes stand for more than the largest float: 240 * 2^120 and 63 * 2^122 are the last below it
    const float most = now >= (FMT == VAMD_KV_E4M3 ? 0x7b800000u : 0x7c800000u) ? (FMT == VAMD_KV_E4M3 ? 240.f : 63.f)
                                                                                : (FMT == VAMD_KV_E4M3 ? 448.f : 127.f);
    auto fit = [&](float v) { return __builtin_amdgcn_fmed3f(v * inv, -most, most); };
    const bool grow = lo > 0 && now != old && !dead;
    // old / new = 2^-(difference of the exponents); beyond 2^-126 every code becomes 0 anyway
    const float ratio = grow && old && now - old < 0x3f800000u ? __uint_as_float(0x3f800000u - (now - old)) : 0.f;
    if (tid == 0 && now != old) *scale = __uint_as_float(now);

    uint8_t* codes = a.codes[kv] + ((int64_t)page * a.heads + h) * a.block * D;
    auto encode_key = [&](const float (&v)[16]) {
        kv_u32x4 w;
#pragma unroll
        for (int e = 0; e < 4; ++e)
            w[e] = dead ? 0u : kv_encode4<FMT>(fit(v[4 * e]), fit(v[4 * e + 1]), fit(v[4 * e + 2]), fit(v[4 * e + 3]));
        return w;
    };
    // codes of four tokens of one feature, from the features' rows
    auto encode_quad = [&](const float (&v)[4][8], int e) {
        return dead ? 0u : kv_encode4<FMT>(fit(v[0][e]), fit(v[1][e]), fit(v[2][e]), fit(v[3][e]));
    };
    auto key_at = [&](int g, int t, int d) { return codes + (int64_t)g * kKvGroup * D + kv_key_at(t & (kKvGroup - 1), d, D); };
    auto quad_at = [&](int g, int p, int gg, int tt) {
        return codes + (int64_t)g * kKvGroup * D + kv_value_at(tt * 16 + gg * 4, p * 8);
    };
    // stores the fresh tokens of a quad (t ..): in a group that is fresh throughout the four lanes of the same features (tiles 0 .. 3) trade
    // dwords, so that each stores the 16 bytes of two features (with 4-byte stores 16 bytes apart 16000 tokens take 28 us where these take 26);
    // else whole dwords, or their bytes beside others that stay
    auto put_quad = [&](uint8_t* to, const float (&v)[4][8], int t) {
        const int group = t & ~(kKvGroup - 1), tt = (t >> 4) & 3;
        if (group >= lo && group + kKvGroup <= hi) {
            uint32_t w[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) w[e] = encode_quad(v, e);
#pragma unroll
            for (int half = 0; half < 2; ++half) {
                kv_u32x4 r = {w[half * 4], w[half * 4 + 1], w[half * 4 + 2], w[half * 4 + 3]};
                kv_transpose_quad(r, tt);
                *(kv_u32x4*)(to - tt * 4 + (half * 4 + tt) * 16) = r;
            }
            return;
        }
        const bool all = t >= lo && t + 4 <= hi;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            const uint32_t c = encode_quad(v, e);
            if (all) *(uint32_t*)(to + e * 16) = c;
            else {
#pragma unroll
                for (int n = 0; n < 4; ++n)
                    if (t + n >= lo && t + n < hi) to[e * 16 + n] = (uint8_t)(c >> (8 * n));
            }
        }
    };
    if (grow) {
        // every other code of the block moves to the new scale (what is fresh is written behind this, by the lanes below)
        const int groups = a.block / kKvGroup;
        if (kv == 0) {
            for (int i = tid; i < groups * pieces; i += nt) {
                int g, t, d;
                key_place(i, g, t, d);
                if (t >= lo && t < hi) continue;
                kv_u32x4* to = (kv_u32x4*)key_at(g, t, d);
                kv_u32x4 w = *to;
#pragma unroll
                for (int e = 0; e < 4; ++e) w[e] = old ? kv_rescale4<FMT>(w[e], ratio) : 0u;
                *to = w;
            }
        } else {
            for (int i = tid; i < groups * quads; i += nt) {
                int g, t, p, gg, tt;
                value_place(i, g, t, p, gg, tt);
                if (t >= lo && t + 4 <= hi) continue;
                uint8_t* to = quad_at(g, p, gg, tt);
#pragma unroll
                for (int e = 0; e < 8; ++e) *(uint32_t*)(to + e * 16) = old ? kv_rescale4<FMT>(*(const uint32_t*)(to + e * 16), ratio) : 0u;
            }
            __syncthreads();                                     // fresh bytes go into these dwords
        }
    }
    if (kv == 0) {
        auto put = [&](int i, const float (&v)[16]) {
            int g, t, d;
            key_place(i + f0 * pieces, g, t, d);
            if (t >= lo && t < hi) *(kv_u32x4*)key_at(g, t, d) = encode_key(v);
        };
        if (held) {
#pragma unroll
            for (int n = 0; n < 2 * HOLD; ++n) {
                float v[16];
#pragma unroll
                for (int e = 0; e < 16; ++e) v[e] = to_f(kept[n >> 1][(n & 1) * 2 * V8 + e / Vec16<T>::N].v[e % Vec16<T>::N]);
                if (tid + n * nt < items) put(tid + n * nt, v);
            }
        } else {
            for (int i = tid; i < items; i += nt) {
                int g, t, d;
                key_place(i + f0 * pieces, g, t, d);
                if (t < lo || t >= hi) continue;
                float v[16], u[2][8];
                kv_load8<T, ALIGNED>(x + t * tok + d, u[0]);
                kv_load8<T, ALIGNED>(x + t * tok + d + 8, u[1]);
#pragma unroll
                for (int e = 0; e < 16; ++e) v[e] = u[e >> 3][e & 7];
                put(i, v);
            }
        }
    } else {
        if (held) {
#pragma unroll
            for (int n = 0; n < HOLD; ++n) {
                float v[4][8];
#pragma unroll
                for (int e = 0; e < 32; ++e) v[e >> 3][e & 7] = to_f(kept[n][e / Vec16<T>::N].v[e % Vec16<T>::N]);
                int g, t, p, gg, tt;
                if (tid + n * nt < items) {
                    value_place(tid + n * nt + f0 * quads, g, t, p, gg, tt);
                    if (t < hi && t + 4 > lo) put_quad(quad_at(g, p, gg, tt), v, t);
                }
            }
        } else {
            for (int i = tid; i < items; i += nt) {
                int g, t, p, gg, tt;
                value_place(i + f0 * quads, g, t, p, gg, tt);
                if (t >= hi || t + 4 <= lo) continue;
                float v[4][8];
#pragma unroll
                for (int n = 0; n < 4; ++n) {
                    if (t + n >= lo && t + n < hi) kv_load8<T, ALIGNED>(x + (t + n) * tok + p * 8, v[n]);
                    else {
#pragma unroll
                        for (int e = 0; e < 8; ++e) v[n][e] = 0.f;
                    }
                }
                put_quad(quad_at(g, p, gg, tt), v, t);
            }
        }
    }
}

// Reading back: one workgroup per (sequence, group of 64 tokens, keys or values, head); a code's value is code * scale, exact.
template <typename T, int FMT, bool ALIGNED>
__global__ void __launch_bounds__(256) kv_read_kernel(const KvIoArgs a) {
    int64_t id = block_number();
    const int h = (int)(id % a.heads);
    id /= a.heads;
    const int kv = (int)(id & 1);
    id >>= 1;
    int j, b;
    if (!kv_io_unit(a, id, kKvGroup, j, b)) return;
    const int64_t start = a.start[b];
    const KvRows rows = kv_rows(a.offsets, b, a.rows, a.most);
    const int64_t base = (start / kKvGroup + j) * kKvGroup;
    const KvSpan span = kv_span(start, rows.count, base, kKvGroup);
    const int lo = span.lo, hi = span.hi;
    if (hi <= lo) return;
    const int page = kv_page(a.table, a.table_stride, a.width, a.blocks, b, base / a.block);
    const bool hole = page < 0;
    const int tid = threadIdx.x, nt = blockDim.x, D = a.D, P = D >> 3;
    const int64_t tok = a.tok[kv], at = hole ? 0 : (int64_t)page * a.heads + h;
    T* y = (T*)a.y[kv] + (rows.first + base - start) * tok + h * a.head[kv];
    const float scale = hole ? 0.f : a.scales[kv][at];
    const uint8_t* codes = a.codes[kv] + (at * a.block + base % a.block) * D;
    if (kv == 0) {
        const int S = D >> 4, pieces = kKvGroup * S;
        for (int q = tid; q < pieces; q += nt) {
            int t, d;
            kv_key_piece(q, S, t, d);
            if (t < lo || t >= hi) continue;
            const kv_u32x4 w = hole ? kv_u32x4{0, 0, 0, 0} : *(const kv_u32x4*)(codes + kv_key_at(t, d, D));
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                const kv_f32x4 l = kv_decode4<FMT>(w[2 * e]), r = kv_decode4<FMT>(w[2 * e + 1]);
                const float v[8] = {l[0] * scale, l[1] * scale, l[2] * scale, l[3] * scale, r[0] * scale, r[1] * scale, r[2] * scale, r[3] * scale};
                kv_store8<T, ALIGNED>(y + t * tok + d + e * 8, v);
            }
        }
    } else {
        for (int q = tid; q < 16 * P; q += nt) {
            const int tt = q & 3, p = (q >> 2) % P, gg = (q >> 2) / P, t = tt * 16 + gg * 4;
            if (t + 4 <= lo || t >= hi) continue;
            const uint8_t* from = codes + kv_value_at(t, p * 8);
            float v[4][8];
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const kv_f32x4 c = kv_decode4<FMT>(hole ? 0u : *(const uint32_t*)(from + e * 16));
#pragma unroll
                for (int n = 0; n < 4; ++n) v[n][e] = c[n] * scale;
            }
#pragma unroll
            for (int n = 0; n < 4; ++n)
                if (t + n >= lo && t + n < hi) kv_store8<T, ALIGNED>(y + (t + n) * tok + p * 8, v[n]);
        }
    }
}

// Arguments that both directions share; returns 0 and fills `a`, or an error.
static int kv_io_args(KvIoArgs& a, const char* name, const void* codes_k, const void* codes_v, const void* scales_k, const void* scales_v,
                      const int32_t* table, int64_t table_stride, const int32_t* start, const int32_t* offsets, int64_t rows, int sequences,
                      int most, int heads, int dim, int block, int width, int blocks, int format, int dtype, int unit, int64_t& grid) {
    VAMD_REQUIRE(sequences > 0 && rows >= 0 && most >= 0 && heads > 0 && heads <= 65536 && width > 0 && blocks > 0 && table_stride >= 0,
                 "%s: bad extents (%d sequences, %lld rows, most %d, %d heads, %d blocks a sequence of %d)", name, sequences, (long long)rows,
                 most, heads, width, blocks);
    VAMD_REQUIRE(dim >= 16 && dim <= 256 && dim % 16 == 0, "%s: dim %d (a multiple of 16, 16 to 256)", name, dim);
    VAMD_REQUIRE(block == 64 || block == 128 || block == 256, "%s: block %d (64, 128 or 256 tokens)", name, block);
    VAMD_REQUIRE(format == VAMD_KV_E4M3 || format == VAMD_KV_INT8, "%s: bad format %d", name, format);
    VAMD_REQUIRE(dtype == VAMD_F32 || dtype == VAMD_BF16, "%s: bad dtype %d", name, dtype);
    VAMD_REQUIRE(codes_k && codes_v && scales_k && scales_v && table && start, "%s: NULL tensor", name);
    VAMD_REQUIRE((uintptr_t)codes_k % 16 == 0 && (uintptr_t)codes_v % 16 == 0 && (uintptr_t)scales_k % 4 == 0 && (uintptr_t)scales_v % 4 == 0 &&
                 (uintptr_t)table % 4 == 0 && (uintptr_t)start % 4 == 0 && (uintptr_t)offsets % 4 == 0, "%s: misaligned tensor", name);
    VAMD_REQUIRE(offsets || rows == (int64_t)sequences * most, "%s: %lld rows are not %d for each of %d sequences", name, (long long)rows, most,
                 sequences);
    a.codes[0] = (uint8_t*)codes_k;
    a.codes[1] = (uint8_t*)codes_v;
    a.scales[0] = (float*)scales_k;
    a.scales[1] = (float*)scales_v;
    a.table = table;
    a.table_stride = table_stride;
    a.start = start;
    a.offsets = offsets;
    a.rows = rows;
    a.sequences = sequences;
    a.heads = heads;
    a.D = dim;
    a.block = block;
    a.width = width;
    a.blocks = blocks;
    a.most = most;
    const KvUnits units = kv_io_units(offsets != nullptr, sequences, rows, most, unit);
    a.touched = units.touched;
    a.listed = units.listed;
    grid = units.count * 2 * heads;
    VAMD_REQUIRE((double)units.count * 2 * heads <= kGridMost, "%s: %d sequences of up to %d rows and %d heads are too many for one call", name, sequences, most, heads);
    return 0;
}
static bool kv_aligned(const KvIoArgs& a, const void* p, const void* q, int dtype) {
    const int n = dtype == VAMD_BF16 ? 8 : 4;
    return (uintptr_t)p % 16 == 0 && (uintptr_t)q % 16 == 0 && a.tok[0] % n == 0 && a.tok[1] % n == 0 && a.head[0] % n == 0 && a.head[1] % n == 0;
}

#define COMMA ,
// KERNEL, which names T, F (format) and A (aligned), for this call's format and alignment; T from VAMD_DISPATCH around it
#define KV_IO_LAUNCH(KERNEL)                                                                                                     \
    do {                                                                                                                         \
        const dim3 g = grid_of(grid), t(threads);                                                                                \
        if (format == VAMD_KV_E4M3) {                                                                                            \
            constexpr int F = VAMD_KV_E4M3;                                                                                      \
            if (aligned) { constexpr bool A = true; hipLaunchKernelGGL((KERNEL), g, t, 0, as_stream(stream), a); }                \
            else { constexpr bool A = false; hipLaunchKernelGGL((KERNEL), g, t, 0, as_stream(stream), a); }                       \
        } else {                                                                                                                 \
            constexpr int F = VAMD_KV_INT8;                                                                                      \
            if (aligned) { constexpr bool A = true; hipLaunchKernelGGL((KERNEL), g, t, 0, as_stream(stream), a); }                \
            else { constexpr bool A = false; hipLaunchKernelGGL((KERNEL), g, t, 0, as_stream(stream), a); }                       \
        }                                                                                                                        \
    } while (0)

}  // namespace vamd

using namespace vamd;

extern "C" int vamd_kv_append(const void* k, int64_t k_token, int64_t k_head, const void* v, int64_t v_token, int64_t v_head,
                              void* codes_k, void* codes_v, float* scales_k, float* scales_v, const int32_t* table, int64_t table_stride,
                              const int32_t* start, const int32_t* offsets, int64_t rows, int sequences, int most, int heads, int dim,
                              int block, int width, int blocks, int format, int dtype, void* stream) {
    KvIoArgs a = {};
    int64_t grid;
    const int rc = kv_io_args(a, "vamd_kv_append", codes_k, codes_v, scales_k, scales_v, table, table_stride, start, offsets, rows, sequences,
                              most, heads, dim, block, width, blocks, format, dtype, block, grid);
    if (rc) return rc;
    if (rows == 0 || most == 0) return 0;
    const int size = dtype == VAMD_BF16 ? 2 : 4;
    VAMD_REQUIRE(k && v && (uintptr_t)k % size == 0 && (uintptr_t)v % size == 0, "vamd_kv_append: NULL or misaligned rows");
    a.x[0] = k;
    a.x[1] = v;
    a.tok[0] = k_token;
    a.tok[1] = v_token;
    a.head[0] = k_head;
    a.head[1] = v_head;
    const bool aligned = kv_aligned(a, k, v, dtype);
    // One wave where a block gets at most 4 tokens (a decoding step: no barrier, more blocks a CU), else four.
    const int threads = most <= 4 ? 64 : 256;
    // What four waves hold in registers: blocks up to 16384 elements (64 or 128 tokens of 128 features) with HOLD 2, up to 32768 with 4
    // (beyond that the rows are read twice).  16000 tokens of 8 heads, 128 features, written and read back in one pass: blocks of 128 tokens
    // 53 us with 2, 66 with 4, 67 read twice; of 256 tokens 60 with 4, 71 read twice.
    if (block * dim <= 16384 || threads == 64) VAMD_DISPATCH(dtype, "vamd_kv_append", KV_IO_LAUNCH(kv_append_kernel<T COMMA F COMMA A COMMA 2>););
    else VAMD_DISPATCH(dtype, "vamd_kv_append", KV_IO_LAUNCH(kv_append_kernel<T COMMA F COMMA A COMMA 4>););
    VAMD_LAUNCH_OK("kv_append");
    return 0;
}

extern "C" int vamd_kv_read(const void* codes_k, const void* codes_v, const float* scales_k, const float* scales_v, const int32_t* table,
                            int64_t table_stride, const int32_t* start, const int32_t* offsets, int64_t rows, int sequences, int most,
                            int heads, int dim, int block, int width, int blocks, int format, void* k, int64_t k_token, int64_t k_head,
                            void* v, int64_t v_token, int64_t v_head, int dtype, void* stream) {
    KvIoArgs a = {};
    int64_t grid;
    const int rc = kv_io_args(a, "vamd_kv_read", codes_k, codes_v, scales_k, scales_v, table, table_stride, start, offsets, rows, sequences,
                              most, heads, dim, block, width, blocks, format, dtype, kKvGroup, grid);
    if (rc) return rc;
    if (rows == 0 || most == 0) return 0;
    const int size = dtype == VAMD_BF16 ? 2 : 4;
    VAMD_REQUIRE(k && v && (uintptr_t)k % size == 0 && (uintptr_t)v % size == 0, "vamd_kv_read: NULL or misaligned rows");
    a.y[0] = k;
    a.y[1] = v;
    a.tok[0] = k_token;
    a.tok[1] = v_token;
    a.head[0] = k_head;
    a.head[1] = v_head;
    const bool aligned = kv_aligned(a, k, v, dtype);
    const int threads = 256;
    VAMD_DISPATCH(dtype, "vamd_kv_read", KV_IO_LAUNCH(kv_read_kernel<T COMMA F COMMA A>););
    VAMD_LAUNCH_OK("kv_read");
    return 0;
}
