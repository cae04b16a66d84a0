// Attention of queries over a cache of 8-bit keys and values (layout, codes and scales: kv_layout.h), paged by a table of
// blocks, for grouped heads, ragged batches, causal with an offset, optionally over a window of the last tokens and a few
// first ones that stay visible:
//
//     s_j = scale * scale_k * (q . code_j) for visible j;   o = sum_j exp(s_j - m) scale_v code_j / sum_j exp(s_j - m)
//
// in one pass over the cache with the running maximum m, sum and output (fp32, exponents in base 2).
//
// kv_attend_rows_kernel: few queries (a decoding step).  A tile is up to 16 rows (query tokens x heads of one key head), so that
// every code of the cache is read once for all heads that share it; bound by reading the cache (64 sequences of up to 4096, 8 key heads
// of 128 features: 56 us, 4.7 TB/s; of 256 features 112, 4.7; float32 queries 63, 4.2).  Each of a workgroup's four
// waves takes every fourth group of 64 tokens of its share of the keys; codes go straight from global memory into MFMA
// operand order (16 bytes a lane, 1 KB a wave and load) and become bf16 in registers: code values are exact there.  With the keys as the
// rows of the first product a lane holds 16 scores of ONE query, and exactly the slots that the second product wants as its
// operand: nothing is exchanged but the row maximum over four lanes.  The next group's keys are loaded behind the first product, its
// values behind the second.  The four waves' partial results meet in LDS; with more than one share per tile
// (long contexts, small batches), they go to the workspace and a second kernel joins them.
//
// float32 queries: a float is the sum of three bf16 numbers, so three products with the exact codes (and three for the
// probabilities) give fp32 accuracy on the same matrix path.
//
// bf16 queries: the codes and the queries are exact, what is rounded are the probabilities (2^-8) on their way into the second product.  With few
// queries they go as two bf16 numbers (2^-16, two products): the result is the formula's but for its own rounding, and the time is
// still that of reading the cache (64 sequences up to 4096 58.3 -> 60.3 us, a window of 2000 25.3 -> 25.6; 16 x 8 queries up to
// 8000 67.8 -> 70.8).  Prompts, bound by the matrix cores, round them once and divide by the sum of the rounded ones: the
// relative error against 64 bits is 0.00182 then, that of the result's rounding alone 0.00165.
#include "kv_layout.h"

#include <type_traits>

namespace vamd {

struct KvAttendArgs {
    const void* q;
    void* o;
    int64_t q_tok, q_head, o_tok, o_head;
    const uint8_t* codes[2];
    const float* scales[2];
    const int32_t* table;
    int64_t table_stride;
    const int32_t* lengths;
    const int32_t* offsets;
    int64_t rows;
    float* part;                 // [tiles of all sequences][heads][tile rows][splits][D] normalised outputs, then [..][splits][2] maximum and sum
    float* part_ml;
    float scale2;                // scale * log2(e)
    int sequences, most, heads, group, D, block_shift, width, blocks, window, sinks, causal, tiles, all_tiles, tile_rows, splits, q_aligned, o_aligned;
};

// Groups of 64 tokens that the rows of a tile can see: `sink_groups` from 0 on, then those from `first` on; `count` in all.
struct KvRange {
    int sink_groups, first, count;
};
__device__ __forceinline__ KvRange kv_range(const KvAttendArgs& a, int length, int p_first, int p_last) {
    int hi = a.causal ? p_last + 1 : length;
    hi = hi > length ? length : hi;
    if (hi <= 0) return KvRange{0, 0, 0};
    const int last = (hi + kKvGroup - 1) / kKvGroup;
    int first = 0, sink = 0;
    if (a.window > 0 && p_first >= a.window) {
        first = (p_first - a.window + 1) / kKvGroup;
        const int s = a.sinks < hi ? a.sinks : hi;
        sink = (s + kKvGroup - 1) / kKvGroup;
        if (sink > first) sink = first;
    }
    return KvRange{sink, first, sink + last - first};
}
// The share of a split: at least 8 groups, so that short sequences of a batch do not fall into crumbs.
// (tiles of many rows: 16 groups, because joining their rows costs more)
__host__ __device__ constexpr int kv_min_share(int tile_rows) { return tile_rows > 16 ? 16 : 8; }
__device__ __forceinline__ int kv_share(int count, int splits, int tile_rows) {
    const int per = (count + splits - 1) / splits, least = kv_min_share(tile_rows);
    return per < least ? least : per;
}
// Rows of a tile that can be there at all.
__host__ __device__ constexpr int kv_tile_fill(int tiles, int tile_rows, int most, int group) { return tiles > 1 ? tile_rows : most * group; }
__device__ __forceinline__ int kv_length(const KvAttendArgs& a, int b) {
    const int64_t room = (int64_t)a.width << a.block_shift;
    int n = a.lengths[b];
    n = n < 0 ? 0 : n;
    return n > room ? (int)room : n;
}

// The sequence of tile number `tile` and the tile's number in it, or false behind the last one.
//
// Only tiles that there are have numbers.  Walked over by `most` instead, the tiles that short sequences do not have lie between the others in a regular pattern that leaves
// whole CUs idle: prompts of 4096 and 925 tokens 435 us, of 4096 alone 264.
__device__ __forceinline__ bool kv_whose_tile(const KvAttendArgs& a, int lane, int& tile, int& b) {
    if (!a.offsets || a.tiles == 1) {
        b = tile / a.tiles;
        tile -= b * a.tiles;
        return b < a.sequences;
    }
    uint32_t number = (uint32_t)tile;
    const bool found = kv_whose(a.sequences, lane, [&](int s) {
        return (kv_rows(a.offsets, s, a.rows, a.most).count * a.group + a.tile_rows - 1) / a.tile_rows;
    }, number, b);
    tile = (int)number;
    return found;
}

__device__ __forceinline__ float kv_over_groups_max(float v) {           // over the four lanes that hold one query's keys
    v = fmaxf(v, __shfl_xor(v, 16, 64));
    return fmaxf(v, __shfl_xor(v, 32, 64));
}
__device__ __forceinline__ float kv_over_groups_sum(float v) {
    v += __shfl_xor(v, 16, 64);
    return v + __shfl_xor(v, 32, 64);
}
// Values up to the largest float.  At a block whose values' scale is above 2^40 (a `big` one) a row's reference goes where the
// probabilities until now (their `sum`, relative to m) come to less than 1/2, and those of this group's 64 keys (up to `top`) to 1/2 at
// most: the output is then no larger than the largest value, whatever the number of keys.  For the same reason results are
// normalised before they are joined, and joined by shares that sum to 1.
constexpr int kKvBig = 40;
__device__ __forceinline__ float kv_big_reference(float m, float sum, float top) {
    return fmaxf(m + (float)((int)(__float_as_uint(sum) >> 23) - 125), top + 7.f);
}
__device__ __forceinline__ float kv_inverse(float l) { return l == 0.f ? 0.f : 1.f / l; }                    // (a row that sees nothing is zero)

__device__ __forceinline__ float kv_finite(float m) { return m == -INFINITY ? 0.f : m; }

// v as the sum of N bf16 numbers, the largest first
template <int N> __device__ __forceinline__ void kv_pieces(float v, bf16_t (&p)[N]) {
#pragma unroll
    for (int i = 0; i < N; ++i) {
        p[i] = (bf16_t)v;
        v -= (float)p[i];
    }
}

// The codes as the loads left them, opaque to the compiler until here: it would convert all of a group's codes where they
// arrive, which takes four times their registers.
__device__ __forceinline__ kv_u32x4 kv_as_loaded(kv_u32x4 w) {
    asm("" : "+v"(w));
    return w;
}

// C: 64-feature chunks of a head (the last one may be partly empty).  ONCE: one tile of rows, so that a sequence's codes are read once, past
// the caches' replacement (256 sequences up to 2000: 117 -> 103 us, 64 of 4160 107 -> 94); with more tiles the others find them there
// (two tiles: 67 us, 71 past it).  Sequences that share the blocks of a common beginning lose nothing by it: 64 of 4160 tokens sharing 4096 49.8 us,
// 49.2 without; 16 of 32832 sharing 32768 90.8, 89.8 without.
template <typename T, int FMT, int C, bool ONCE>
__global__ void __launch_bounds__(256, C <= 2 ? 2 : 1) kv_attend_rows_kernel(const KvAttendArgs a) {
    constexpr int N = sizeof(T) == 4 ? 3 : 1, PN = sizeof(T) == 4 ? 3 : 2;       // bf16 pieces of a query, of a probability
    extern __shared__ __attribute__((aligned(16))) float lds[];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int r = lane & 15, g = lane >> 4;
    // Heads vary fastest, then the tiles, shares slowest: workgroups without work (shares that a short sequence does not have) then sit
    // behind each other and not on every second XCD or CU.
    uint32_t id = block_number();
    const int h = (int)(id % (uint32_t)a.heads);
    id /= (uint32_t)a.heads;
    const uint32_t tiles = (uint32_t)a.all_tiles;
    const int split = (int)(id / tiles);
    if (split >= a.splits) return;
    int tile = (int)(id % tiles), b;
    const int64_t slot = ((int64_t)tile * a.heads + h) * 16;
    if (ONCE) {
        b = tile;
        tile = 0;
    } else if (!kv_whose_tile(a, lane, tile, b)) return;

    const KvRows rows = kv_rows(a.offsets, b, a.rows, a.most);
    if (tile * 16 >= rows.count * a.group) return;
    const int length = kv_length(a, b);
    const int shift = length - (int)rows.all;                               // position of the sequence's first query
    const int row = tile * 16 + r, tok = row / a.group;
    const bool live = tok < rows.count;
    const int pos = a.causal ? shift + tok : length - 1;
    int last_row = tile * 16 + 15;
    last_row = last_row < rows.count * a.group ? last_row : rows.count * a.group - 1;
    const int p_first = a.causal ? shift + tile * 16 / a.group : length - 1, p_last = a.causal ? shift + last_row / a.group : length - 1;
    const KvRange range = kv_range(a, length, p_first, p_last);
    const int per = kv_share(range.count, a.splits, a.tile_rows);
    const int begin = split * per, end = begin + per < range.count ? begin + per : range.count;
    if (split > 0 && begin >= range.count) return;

    const int head = h * a.group + row - tok * a.group;
    const int S = a.D >> 4;
    // the queries' loads are issued before the first keys' and taken apart behind them
    Vec16<T> q_raw[C * 2][8 / Vec16<T>::N];
    {
        const T* q = (const T*)a.q + (rows.first + (live ? tok : 0)) * a.q_tok + head * a.q_head;
#pragma unroll
        for (int c = 0; c < C * 2; ++c) {
            const int d = (c >> 1) * 64 + g * 16 + (c & 1) * 8;
#pragma unroll
            for (int i = 0; i < 8 / Vec16<T>::N; ++i) {
                q_raw[c][i] = Vec16<T>{};
                if (live && d < a.D) {
                    const T* p = q + d + i * Vec16<T>::N;
                    if (a.q_aligned) q_raw[c][i] = *(const Vec16<T>*)p;
                    else {
#pragma unroll
                        for (int e = 0; e < Vec16<T>::N; ++e) q_raw[c][i].v[e] = p[e];
                    }
                }
            }
        }
    }

    kv_f32x4 acc[C * 4];
#pragma unroll
    for (int t = 0; t < C * 4; ++t) acc[t] = kv_f32x4{0.f, 0.f, 0.f, 0.f};
    float m = -INFINITY, l = 0.f;

    // The group with running number x: its block (block 0 in place of a hole, none of whose tokens is seen), its bytes.
    auto group_of = [&](int x) { return x < range.sink_groups ? x : x - range.sink_groups + range.first; };
    auto page_of = [&](int x) {
        return x < end ? kv_page(a.table, a.table_stride, a.width, a.blocks, b, group_of(x) >> (a.block_shift - 6)) : -1;
    };
    auto at_of = [&](int page) { return (int64_t)(page < 0 ? 0 : page) * a.heads + h; };
    auto bytes_of = [&](int kv, int page, int x) {
        const int in_block = group_of(x) & ((1 << (a.block_shift - 6)) - 1);
        return a.codes[kv] + ((at_of(page) << a.block_shift) + in_block * kKvGroup) * a.D;
    };
    auto load = [](const uint8_t* p) { return ONCE ? __builtin_nontemporal_load((const kv_u32x4*)p) : *(const kv_u32x4*)p; };
    kv_u32x4 kc[4 * C], vc[4 * C];
    float ks = 0.f, vs = 0.f;
    // in a last chunk that the head does not fill, lanes without a slab read the chunk's first one: their queries are zero
    const int k_lane = lane * 16, k_lane_last = ((C - 1) * 4 + g < S ? lane : r) * 16;
    auto load_k = [&](int page, int x) {
        const uint8_t* p = bytes_of(0, page, x);
        ks = a.scales[0][at_of(page)];
#pragma unroll
        for (int t = 0; t < 4; ++t)
#pragma unroll
            for (int c = 0; c < C; ++c) kc[t * C + c] = load(p + kv_key_at(t * 16, c * 64, a.D) + (c < C - 1 ? k_lane : k_lane_last));
    };
    auto load_v = [&](int page, int x) {
        const uint8_t* p = bytes_of(1, page, x);
        vs = a.scales[1][at_of(page)];
#pragma unroll
        for (int s = 0; s < 4 * C; ++s)
            if (s < S) vc[s] = load(p + kv_value_at(0, s * 16) + k_lane);
    };
    int x = begin + wave;
    int page = page_of(x), next = page_of(x + 4);
    if (x < end) {
        load_k(page, x);
        load_v(page, x);
    }
    kv_bf16x8 qf[N][C * 2];
#pragma unroll
    for (int c = 0; c < C * 2; ++c)
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            const T v = q_raw[c][e / Vec16<T>::N].v[e % Vec16<T>::N];
            if constexpr (N == 1) qf[0][c][e] = v;
            else {
                bf16_t p[N];
                kv_pieces<N>(v, p);
#pragma unroll
                for (int n = 0; n < N; ++n) qf[n][c][e] = p[n];
            }
        }
    // what this lane's query sees: keys up to `upto`, from `from` on or below `first_keys`
    const int upto = pos < length ? pos : length - 1, from = a.window > 0 ? pos - a.window + 1 : 0, first_keys = a.window > 0 ? a.sinks : 0;
    for (; x < end; x += 4) {
        const int after = page_of(x + 8);
        const bool more = x + 4 < end;
        kv_f32x4 sc[4];
#pragma unroll
        for (int t = 0; t < 4; ++t) {
            sc[t] = kv_f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int c = 0; c < C; ++c) {
                const kv_u32x4 w = kv_as_loaded(kc[t * C + c]);
#pragma unroll
                for (int u = 0; u < 2; ++u) {
                    const kv_bf16x8 kf = kv_operand8<FMT>(w[u * 2], w[u * 2 + 1]);
#pragma unroll
                    for (int n = N - 1; n >= 0; --n) sc[t] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(kf, qf[n][c * 2 + u], sc[t], 0, 0, 0);
                }
            }
            __builtin_amdgcn_sched_barrier(0);
        }
        const float f = a.scale2 * ks, v_scale = vs;
        const int k0 = group_of(x) * kKvGroup;
        if (more) load_k(next, x + 4);
        // keys that some row of the tile does not see?
        const bool edge = page < 0 || k0 + kKvGroup > p_first + 1 || k0 + kKvGroup > length ||
                          (a.window > 0 && k0 <= p_last - a.window && k0 + kKvGroup > a.sinks);
#pragma unroll
        for (int t = 0; t < 4; ++t)
#pragma unroll
            for (int i = 0; i < 4; ++i) sc[t][i] *= f;
        if (edge) {
            const int k_lane0 = k0 + g * 4;
            const int rel_upto = page < 0 ? -1 : upto - k_lane0, rel_from = from - k_lane0, rel_first = first_keys - k_lane0;
#pragma unroll
            for (int t = 0; t < 4; ++t)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const int j = t * 16 + i;
                    const bool seen = j <= rel_upto && (j >= rel_from || j < rel_first);
                    sc[t][i] = seen ? sc[t][i] : -INFINITY;
                }
        }
        float top = -INFINITY;
#pragma unroll
        for (int t = 0; t < 4; ++t)
#pragma unroll
            for (int i = 0; i < 4; ++i) top = fmaxf(top, sc[t][i]);
        top = kv_over_groups_max(top);
        float m_new = fmaxf(m, top);
        if ((int)(__float_as_uint(v_scale) >> 23) - 127 > kKvBig) m_new = kv_big_reference(m, kv_over_groups_sum(l), top);
        const float m_use = kv_finite(m_new);
        if (__any(m_new != m)) {
            const float alpha = __builtin_amdgcn_exp2f(m - m_use);
            l *= alpha;
#pragma unroll
            for (int t = 0; t < C * 4; ++t)
#pragma unroll
                for (int i = 0; i < 4; ++i) acc[t][i] *= alpha;
        }
        m = m_new;
#pragma unroll
        for (int t = 0; t < 4; ++t)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const float e = __builtin_amdgcn_exp2f(sc[t][i] - m_use);
                l += e;
                sc[t][i] = e * v_scale;          // the values' scale goes into the probability: a power of two, nothing is rounded
            }
        if (v_scale != v_scale) {                // a block that reads as NaN is NaN only to the queries that see it
#pragma unroll
            for (int t = 0; t < 4; ++t)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const int j = k0 + t * 16 + g * 4 + i;
                    const bool seen = page >= 0 && j <= upto && (j >= from || j < first_keys);
                    sc[t][i] = seen ? sc[t][i] : 0.f;
                }
        }
        kv_bf16x8 pf[PN][2];
#pragma unroll
        for (int t = 0; t < 4; ++t)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                bf16_t p[PN];
                kv_pieces<PN>(sc[t][i], p);
#pragma unroll
                for (int n = 0; n < PN; ++n) pf[n][t >> 1][(t & 1) * 4 + i] = p[n];
            }
#pragma unroll
        for (int s = 0; s < C * 4; ++s) {
            if (s < S) {
                const kv_u32x4 w = kv_as_loaded(vc[s]);
#pragma unroll
                for (int u = 0; u < 2; ++u) {
                    const kv_bf16x8 vf = kv_operand8<FMT>(w[u * 2], w[u * 2 + 1]);
#pragma unroll
                    for (int n = PN - 1; n >= 0; --n) acc[s] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(vf, pf[n][u], acc[s], 0, 0, 0);
                }
            }
            __builtin_amdgcn_sched_barrier(0);
        }
        if (more) load_v(next, x + 4);
        page = next;
        next = after;
    }
    l = kv_over_groups_sum(l);
    {
        const float inv = kv_inverse(l);
#pragma unroll
        for (int t = 0; t < C * 4; ++t)
#pragma unroll
            for (int i = 0; i < 4; ++i) acc[t][i] *= inv;
    }

    // the four waves' results: 2 and 3 hand theirs to 0 and 1, then 1 to 0
    float* box_ml = lds + 2 * 64 * C * 16;
#pragma unroll
    for (int step = 2; step > 0; step >>= 1) {
        if (wave >= step && wave < 2 * step) {
            float* box = lds + (wave - step) * 64 * C * 16;
#pragma unroll
            for (int t = 0; t < C * 4; ++t) *(kv_f32x4*)(box + (t * 64 + lane) * 4) = acc[t];
            box_ml[((wave - step) * 64 + lane) * 2] = m;
            box_ml[((wave - step) * 64 + lane) * 2 + 1] = l;
        }
        __syncthreads();
        if (wave < step) {
            const float* box = lds + wave * 64 * C * 16;
            const float m2 = box_ml[(wave * 64 + lane) * 2], l2 = box_ml[(wave * 64 + lane) * 2 + 1];
            const float m_new = fmaxf(m, m2), m_use = kv_finite(m_new);
            const float w1 = l * __builtin_amdgcn_exp2f(m - m_use), w2 = l2 * __builtin_amdgcn_exp2f(m2 - m_use);
            m = m_new;
            l = w1 + w2;
            const float inv = kv_inverse(l), f1 = w1 * inv, f2 = w2 * inv;
#pragma unroll
            for (int t = 0; t < C * 4; ++t) {
                const kv_f32x4 o = *(const kv_f32x4*)(box + (t * 64 + lane) * 4);
#pragma unroll
                for (int i = 0; i < 4; ++i) acc[t][i] = acc[t][i] * f1 + o[i] * f2;
            }
        }
        __syncthreads();
    }
    if (wave > 0 || !live) return;
    if (a.splits > 1) {
        float* part = a.part + ((slot + r) * a.splits + split) * a.D;
#pragma unroll
        for (int t = 0; t < C * 4; ++t)
            if (t < S) *(kv_f32x4*)(part + t * 16 + g * 4) = acc[t];
        if (g == 0) {
            float* ml = a.part_ml + ((slot + r) * a.splits + split) * 2;
            ml[0] = m;
            ml[1] = l;
        }
        return;
    }
    T* o = (T*)a.o + (rows.first + tok) * a.o_tok + head * a.o_head;
#pragma unroll
    for (int t = 0; t < C * 4; ++t) {
        if (t >= S) continue;
        T v[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) v[i] = from_f<T>(acc[t][i]);
        if (a.o_aligned) {
            if (sizeof(T) == 4) *(kv_u32x4*)(o + t * 16 + g * 4) = *(const kv_u32x4*)v;
            else *(kv_u32x2*)(o + t * 16 + g * 4) = *(const kv_u32x2*)v;
        } else {
#pragma unroll
            for (int i = 0; i < 4; ++i) o[t * 16 + g * 4 + i] = v[i];
        }
    }
}

// ---------------------------------------------------------------------------------------------------- many queries (prompts)
//
// A workgroup of four waves takes 128 rows, a wave 32 of them as the columns of v_mfma_f32_32x32x16_bf16, and walks over the keys 64 at
// a time (KW = 1); or 64 rows, two waves on each half of the keys (KW = 2), whose results meet in LDS at the end: half
// the time for a tile where there are few of them.  The codes of a group become bf16 ONCE per workgroup on their way into LDS (both
// operands in the order in which the products read them, 16 bytes a lane, no bank conflicts; the next group's codes are in
// flight meanwhile and go to the other buffer behind the products, one barrier a group).  A lane ends up with 16 scores of
// one query per 32 keys, again in the slots in which the second product wants the probabilities: the row maximum needs
// one exchange between two lanes.  The running maximum is a reference that moves only when a score exceeds it by 2^8 or more
// (probabilities up to 256 are as exact as below 1), so that the outputs are hardly ever rescaled.  The values' power-of-two
// scale goes into the exponent.
//
// Bound by the matrix cores, the exponentials and the LDS reads about alike (an operand is read once for 32 queries, 128 bytes a
// clock): 30000 keys before 2048 queries of 32 heads, 128 features, 940 TFLOP/s; prompts of 4096 and 925 tokens behind
// 1000 714 (kernel trace, 301 us) to 818 (passes in a row, 263 us), where causal tiles of unlike length leave some of the chip idle; a
// plain bf16 product of 8192^3 reaches 1234.
//
// DT: tiles of 32 features (the last may be half empty).
__device__ __forceinline__ float kv_over_halves_max(float v) {               // over the two lanes that hold one query's keys
    const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
__device__ __forceinline__ float kv_over_halves_sum(float v) {
    const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}

constexpr int kKvTileThreads = 256;

template <typename T, int FMT, int DT, int KW>
__global__ void __launch_bounds__(kKvTileThreads, DT <= (sizeof(T) == 4 ? 2 : 4) ? 2 : 1) kv_attend_tile_kernel(const KvAttendArgs a) {
    constexpr int N = sizeof(T) == 4 ? 3 : 1;
    constexpr int PIECES = (DT * 2 * 64 + kKvTileThreads - 1) / kKvTileThreads;      // 16-byte pieces of a group a thread stages
    constexpr int KBYTES = DT * 4 * 64 * 16, BUF = 2 * KBYTES;
    constexpr int KH = 2 / KW, ROW_WAVES = 4 / KW;                           // halves of a group's keys a wave takes; waves over the rows
    extern __shared__ __attribute__((aligned(16))) unsigned char smem[];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int c = lane & 31, hh = lane >> 5, wave_r = wave % ROW_WAVES, kh0 = wave / ROW_WAVES;
    // Heads vary fastest (where they are a multiple of 8 the tiles of one meet in one XCD's L2), then the shares, then the tiles, late
    // ones of a sequence (the longest, where queries are causal) first.
    uint32_t id = block_number();
    const int h = (int)(id % (uint32_t)a.heads);
    id /= (uint32_t)a.heads;
    const int split = (int)(id % (uint32_t)a.splits);
    int tile = (int)(id / (uint32_t)a.splits), b;
    if (tile >= a.all_tiles) return;
    const int64_t slot = ((int64_t)tile * a.heads + h) * a.tile_rows;
    if (!kv_whose_tile(a, lane, tile, b)) return;
    const KvRows rows = kv_rows(a.offsets, b, a.rows, a.most);
    const int all_rows = rows.count * a.group;
    tile = (all_rows + a.tile_rows - 1) / a.tile_rows - 1 - tile;
    if (tile < 0) return;
    const int first_row = tile * a.tile_rows;
    const int length = kv_length(a, b), shift = length - (int)rows.all;
    const int last_row = first_row + a.tile_rows - 1 < all_rows ? first_row + a.tile_rows - 1 : all_rows - 1;
    const int p_first = a.causal ? shift + first_row / a.group : length - 1, p_last = a.causal ? shift + last_row / a.group : length - 1;
    const KvRange range = kv_range(a, length, p_first, p_last);
    const int per = kv_share(range.count, a.splits, a.tile_rows);
    const int begin = split * per, end = begin + per < range.count ? begin + per : range.count;
    if (split > 0 && begin >= range.count) return;
    const int S = a.D >> 4;

    auto group_of = [&](int x) { return x < range.sink_groups ? x : x - range.sink_groups + range.first; };
    // The table's entries and the scales come through vector loads (an address that depends on a register): a scalar load in
    // flight makes every wait for LDS a wait for all of it.  Entries are loaded two groups ahead.
    int lane_zero;
    asm volatile("v_mov_b32 %0, 0" : "=v"(lane_zero));
    const int32_t* entries = a.table + b * a.table_stride + lane_zero;
    auto entry_of = [&](int x) {                             // length <= width blocks: never behind the table's row
        x = x < end ? x : end - 1;
        return entries[group_of(x) >> (a.block_shift - 6)];
    };
    kv_u32x4 st[2][PIECES];                                                  // codes of the group after this one
    float ks_next = 0.f, vs_next = 0.f;
    int page_next = -1, entry = -1;
    auto fetch = [&](int x) {
        page_next = __builtin_amdgcn_readfirstlane(entry);
        if (page_next >= a.blocks) page_next = -1;           // a hole, as a negative entry is
        const int64_t at = (int64_t)(page_next < 0 ? 0 : page_next) * a.heads + h;
        const int64_t byte = ((at << a.block_shift) + (group_of(x) & ((1 << (a.block_shift - 6)) - 1)) * kKvGroup) * a.D;
#pragma unroll
        for (int i = 0; i < PIECES; ++i) {
            const int q = tid + i * kKvTileThreads;
            if (q < 64 * S) {
                st[0][i] = *((const kv_u32x4*)(a.codes[0] + byte) + q);
                st[1][i] = *((const kv_u32x4*)(a.codes[1] + byte) + q);
            }
        }
        ks_next = (a.scales[0] + at)[lane_zero];
        vs_next = (a.scales[1] + at)[lane_zero];
        entry = entry_of(x + 1);
    };
    // keys: [8 features][64 tokens]; values: [step of 16 tokens][half][feature], 8 tokens each (see above)
    auto stage = [&](int buf) {
        unsigned char* kb = smem + buf * BUF;
        unsigned char* vb = kb + KBYTES;
#pragma unroll
        for (int i = 0; i < PIECES; ++i) {
            const int q = tid + i * kKvTileThreads;
            if (q < 64 * S) {
                int token, kd, g, d;
                kv_key_piece(q, S, token, kd);
                kv_value_piece(q, g, d);
                const kv_u32x4 kw = kv_as_loaded(st[0][i]);
                *(kv_bf16x8*)(kb + ((kd >> 3) * 64 + token) * 16) = kv_operand8<FMT>(kw[0], kw[1]);
                *(kv_bf16x8*)(kb + ((kd >> 3) * 64 + 64 + token) * 16) = kv_operand8<FMT>(kw[2], kw[3]);
                if (FMT == VAMD_KV_INT8) __builtin_amdgcn_sched_barrier(0);  // one conversion's floats at a time
                const kv_u32x4 vw = kv_as_loaded(st[1][i]);
#pragma unroll
                for (int u = 0; u < 2; ++u) {
                    const kv_bf16x8 w = kv_operand8<FMT>(vw[2 * u], vw[2 * u + 1]);
                    const kv_u32x4 bits = __builtin_bit_cast(kv_u32x4, w);
                    unsigned char* to = vb + (((4 * u + (g & 1)) * (DT * 32)) + d) * 16 + (g >> 1) * 8;
                    *(kv_u32x2*)to = kv_u32x2{bits[0], bits[1]};
                    *(kv_u32x2*)(to + 2 * (DT * 32) * 16) = kv_u32x2{bits[2], bits[3]};
                    if (FMT == VAMD_KV_INT8) __builtin_amdgcn_sched_barrier(0);
                }
            }
        }
    };

    if (begin < end) {
        entry = entry_of(begin);
        fetch(begin);
    }
    // queries: column c is row first_row + 32 wave_r + c
    const int row = first_row + wave_r * 32 + c, tok = row / a.group, head = h * a.group + row - tok * a.group;
    const bool live = tok < rows.count;
    const int pos = a.causal ? shift + tok : length - 1;
    const int upto = pos < length ? pos : length - 1, from = a.window > 0 ? pos - a.window + 1 : 0, first_keys = a.window > 0 ? a.sinks : 0;
    kv_bf16x8 qf[N][DT * 2];
    {
        const T* q = (const T*)a.q + (rows.first + (live ? tok : 0)) * a.q_tok + head * a.q_head;
#pragma unroll
        for (int k = 0; k < DT * 2; ++k) {
            T v[8] = {};
            if (live && k < S) {
                const T* p = q + k * 16 + hh * 8;
                if (a.q_aligned) {
#pragma unroll
                    for (int i = 0; i < 8 / Vec16<T>::N; ++i) *(Vec16<T>*)(v + i * Vec16<T>::N) = *(const Vec16<T>*)(p + i * Vec16<T>::N);
                } else {
#pragma unroll
                    for (int e = 0; e < 8; ++e) v[e] = p[e];
                }
            }
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                if constexpr (N == 1) qf[0][k][e] = v[e];
                else {
                    bf16_t p[N];
                    kv_pieces<N>(v[e], p);
#pragma unroll
                    for (int n = 0; n < N; ++n) qf[n][k][e] = p[n];
                }
            }
        }
    }
    kv_f32x16 acc[DT];
    float m = -INFINITY, l = 0.f;
#pragma unroll
    for (int t = 0; t < DT; ++t)
#pragma unroll
        for (int i = 0; i < 16; ++i) acc[t][i] = 0.f;
    if (begin < end) {
        // keys' slabs that the head does not have are zero in both buffers (values' rows there end up in outputs that nobody reads)
        for (int q = S * 128 + tid; q < DT * 2 * 128; q += kKvTileThreads) {
            *(kv_u32x4*)(smem + q * 16) = kv_u32x4{0, 0, 0, 0};
            *(kv_u32x4*)(smem + BUF + q * 16) = kv_u32x4{0, 0, 0, 0};
        }
        stage(0);
    }
    int buf = 0;
    for (int x = begin; x < end; ++x, buf ^= 1) {
        const float f_raw = a.scale2 * __uint_as_float(__builtin_amdgcn_readfirstlane(__float_as_uint(ks_next)));
        const float v_scale = __uint_as_float(__builtin_amdgcn_readfirstlane(__float_as_uint(vs_next)));
        const int page = page_next, k0 = group_of(x) * kKvGroup;
        const bool more = x + 1 < end;
        __syncthreads();                                     // this buffer is written, the other one read
        if (more) fetch(x + 1);
        const unsigned char* kb = smem + buf * BUF;
        const unsigned char* vb = kb + KBYTES;
        // operands are read in batches of R, one batch ahead of the products
        constexpr int READS = KH * 2 * DT, R = READS % 4 ? 2 : 4, BATCHES = READS / R;
        kv_bf16x8 fr[2][R];
        auto read_k = [&](int i) {                           // batch i: keys 32 (kh0 + kh) + c, features 16 k + 8 hh ..
#pragma unroll
            for (int e = 0; e < R; ++e) {
                const int kh = (i * R + e) / (DT * 2), k = (i * R + e) % (DT * 2);
                fr[i & 1][e] = *(const kv_bf16x8*)(kb + ((k * 2 + hh) * 64 + (kh0 + kh) * 32 + c) * 16);
            }
        };
        auto read_v = [&](int i) {                           // batch i: feature 32 t + c, tokens of step s and half hh
#pragma unroll
            for (int e = 0; e < R; ++e) {
                const int s = (i * R + e) / DT, t = (i * R + e) % DT;
                fr[i & 1][e] = *(const kv_bf16x8*)(vb + (((kh0 * 2 + s) * 2 + hh) * (DT * 32) + t * 32 + c) * 16);
            }
        };
        kv_f32x16 sc[KH];
#pragma unroll
        for (int kh = 0; kh < KH; ++kh)
#pragma unroll
            for (int i = 0; i < 16; ++i) sc[kh][i] = 0.f;
        read_k(0);
#pragma unroll
        for (int i = 0; i < BATCHES; ++i) {
            if (i + 1 < BATCHES) read_k(i + 1);
#pragma unroll
            for (int e = 0; e < R; ++e) {
                const int kh = (i * R + e) / (DT * 2), k = (i * R + e) % (DT * 2);
#pragma unroll
                for (int n = N - 1; n >= 0; --n) sc[kh] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(fr[i & 1][e], qf[n][k], sc[kh], 0, 0, 0);
            }
            __builtin_amdgcn_sched_barrier(0);
        }
        read_v(0);                                           // in flight during the softmax
        // scores stay unscaled until the exponential, which takes a positive factor; any other one (negative, 0, NaN) is applied here
        const bool by_hand = !(f_raw > 0.f && f_raw < INFINITY);
        const float f = by_hand ? 1.f : f_raw;
        if (by_hand) {
#pragma unroll
            for (int kh = 0; kh < KH; ++kh)
#pragma unroll
                for (int i = 0; i < 16; ++i) sc[kh][i] *= f_raw;
        }
        const bool edge = page < 0 || k0 + kKvGroup > p_first + 1 || k0 + kKvGroup > length ||
                          (a.window > 0 && k0 <= p_last - a.window && k0 + kKvGroup > a.sinks);
        // 2^e = v_scale is added to the exponents unless it is so far from 1 that probabilities could leave the range of a float
        const int v_exp = (int)(__float_as_uint(v_scale) >> 23) - 127;
        const bool fold = v_exp >= -40 && v_exp <= kKvBig;
        const float v_add = fold ? (float)v_exp : 0.f, v_undo = fold ? __uint_as_float((uint32_t)(127 - v_exp) << 23) : 1.f;
        const int k1 = k0 + kh0 * 32 + hh * 4;               // token of the lane's first score
        if (edge) {
            const int rel_upto = page < 0 ? -1 : upto - k1, rel_from = from - k1, rel_first = first_keys - k1;
#pragma unroll
            for (int kh = 0; kh < KH; ++kh)
#pragma unroll
                for (int i = 0; i < 16; ++i) {
                    const int j = kh * 32 + (i >> 2) * 8 + (i & 3);
                    const bool seen = j <= rel_upto && (j >= rel_from || j < rel_first);
                    sc[kh][i] = seen ? sc[kh][i] : -INFINITY;
                }
        }
        float top = -INFINITY;
#pragma unroll
        for (int kh = 0; kh < KH; ++kh)
#pragma unroll
            for (int i = 0; i < 16; ++i) top = fmaxf(top, sc[kh][i]);
        top = kv_over_halves_max(top) * f;
        const bool big = v_exp > kKvBig;
        if (__any(top > m + 8.f) || big) {
            const float m_new = big ? kv_big_reference(m, kv_over_halves_sum(l), top) : top > m + 8.f ? top : m;
            const float alpha = __builtin_amdgcn_exp2f(m - kv_finite(m_new));
            l *= alpha;
#pragma unroll
            for (int t = 0; t < DT; ++t)
#pragma unroll
                for (int i = 0; i < 16; ++i) acc[t][i] *= alpha;
            m = m_new;
        }
        const float shift_by = v_add - kv_finite(m);
        float sum = 0.f;
#pragma unroll
        for (int kh = 0; kh < KH; ++kh)
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                const float e = __builtin_amdgcn_exp2f(fmaf(sc[kh][i], f, shift_by));
                if (N > 1) sum += e;
                sc[kh][i] = e;
            }
        kv_bf16x8 pf[N][2 * KH];
        auto take_apart = [&]() {
#pragma unroll
            for (int s = 0; s < 2 * KH; ++s)
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    bf16_t p[N];
                    kv_pieces<N>(sc[s >> 1][(s & 1) * 8 + e], p);
#pragma unroll
                    for (int n = 0; n < N; ++n) pf[n][s][e] = p[n];
                }
        };
        take_apart();
        if (N == 1) {
            // the sum of the probabilities as they are multiplied, rounded: the rounding of a key that dominates a row then cancels in the
            // quotient (error against 64 bits behind 700 keys: 0.00204 -> 0.00183; the rounding of the result alone is 0.00165)
            const kv_bf16x2 ones = {(bf16_t)1.f, (bf16_t)1.f};
#pragma unroll
            for (int s = 0; s < 2 * KH; ++s)
#pragma unroll
                for (int e = 0; e < 8; e += 2)
                    sum = __builtin_amdgcn_fdot2_f32_bf16(kv_bf16x2{pf[0][s][e], pf[0][s][e + 1]}, ones, sum, false);
        }
        l = fmaf(sum, v_undo, l);
        if (!fold) {                                         // NaN: only to the queries that see the block
#pragma unroll
            for (int kh = 0; kh < KH; ++kh)
#pragma unroll
                for (int i = 0; i < 16; ++i) {
                    const int j = k1 + kh * 32 + (i >> 2) * 8 + (i & 3);
                    const bool seen = page >= 0 && j <= upto && (j >= from || j < first_keys);
                    sc[kh][i] = seen ? sc[kh][i] * v_scale : 0.f;
                }
            take_apart();
        }
#pragma unroll
        for (int i = 0; i < BATCHES; ++i) {
            if (i + 1 < BATCHES) read_v(i + 1);
#pragma unroll
            for (int e = 0; e < R; ++e) {
                const int s = (i * R + e) / DT, t = (i * R + e) % DT;
#pragma unroll
                for (int n = N - 1; n >= 0; --n) acc[t] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(fr[i & 1][e], pf[n][s], acc[t], 0, 0, 0);
            }
            __builtin_amdgcn_sched_barrier(0);
        }
        if (more) stage(buf ^ 1);
    }
    float total = kv_over_halves_sum(l), inv = kv_inverse(total);
    if constexpr (KW == 2) {
        // the waves of the keys' second halves hand theirs to those of the first: [wave_r][register][lane]
        __syncthreads();
        float* box = (float*)smem + wave_r * (DT * 16 + 2) * 64 + lane;
        if (kh0 == 1) {
#pragma unroll
            for (int t = 0; t < DT; ++t)
#pragma unroll
                for (int i = 0; i < 16; ++i) box[(t * 16 + i) * 64] = acc[t][i] * inv;
            box[DT * 16 * 64] = m;
            box[(DT * 16 + 1) * 64] = total;
        }
        __syncthreads();
        if (kh0 == 1) return;
        const float m2 = box[DT * 16 * 64], m_new = fmaxf(m, m2);
        const float w1 = __builtin_amdgcn_exp2f(m - kv_finite(m_new));
        const float w2 = box[(DT * 16 + 1) * 64] * __builtin_amdgcn_exp2f(m2 - kv_finite(m_new));
        m = m_new;
        total = total * w1 + w2;
        inv = kv_inverse(total);
        const float f1 = w1 * inv, f2 = w2 * inv;            // (this wave's output is not normalised yet, the other's is)
#pragma unroll
        for (int t = 0; t < DT; ++t)
#pragma unroll
            for (int i = 0; i < 16; ++i) acc[t][i] = acc[t][i] * f1 + box[(t * 16 + i) * 64] * f2;
        inv = 1.f;
    }
    if (!live) return;
    if (a.splits > 1) {
        const int64_t at = (slot + wave_r * 32 + c) * a.splits + split;
        float* part = a.part + at * a.D;
#pragma unroll
        for (int t = 0; t < DT; ++t)
#pragma unroll
            for (int i = 0; i < 4; ++i)
                if (t * 2 + (i >> 1) < S)
                    *(kv_f32x4*)(part + t * 32 + i * 8 + hh * 4) =
                        kv_f32x4{acc[t][4 * i] * inv, acc[t][4 * i + 1] * inv, acc[t][4 * i + 2] * inv, acc[t][4 * i + 3] * inv};
        if (hh == 0) {
            a.part_ml[at * 2] = m;
            a.part_ml[at * 2 + 1] = total;
        }
        return;
    }
    T* o = (T*)a.o + (rows.first + tok) * a.o_tok + head * a.o_head;
#pragma unroll
    for (int t = 0; t < DT; ++t)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            if (t * 2 + (i >> 1) >= S) continue;
            T v[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) v[e] = from_f<T>(acc[t][4 * i + e] * inv);
            T* to = o + t * 32 + i * 8 + hh * 4;
            if (a.o_aligned) {
                if (sizeof(T) == 4) *(kv_u32x4*)to = *(const kv_u32x4*)v;
                else *(kv_u32x2*)to = *(const kv_u32x2*)v;
            } else {
#pragma unroll
                for (int e = 0; e < 4; ++e) to[e] = v[e];
            }
        }
}

// Joins the shares of a row: one workgroup of 16 waves per row.  The shares' weights go to LDS first, so that the loads of the
// outputs depend on nothing; a lane then reads four features of every (1024 / lanes a row takes)-th share, eight in flight.
constexpr int kKvMaxSplits = 256;
template <typename T, int kKvJoin>
__global__ void __launch_bounds__(kKvJoin) kv_join_kernel(const KvAttendArgs a) {
    __shared__ float weight[kKvMaxSplits], box_m[4], box_l[4];
    __shared__ __attribute__((aligned(16))) float box[kKvJoin * 4];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    uint32_t id = blockIdx.x;
    const uint32_t per_tile = (uint32_t)kv_tile_fill(a.tiles, a.tile_rows, a.most, a.group);
    int row = (int)(id % per_tile);
    id /= per_tile;
    const int64_t slot = (int64_t)id * a.tile_rows + row;
    const int h = (int)(id % (uint32_t)a.heads);
    int tile = (int)(id / (uint32_t)a.heads), b;
    if (!kv_whose_tile(a, lane, tile, b)) return;
    const KvRows rows = kv_rows(a.offsets, b, a.rows, a.most);
    if (a.tile_rows > 16) tile = (rows.count * a.group + a.tile_rows - 1) / a.tile_rows - 1 - tile;      // the tile kernel's order
    row += tile * a.tile_rows;
    const int tok = row / a.group;
    if (tile < 0 || tok >= rows.count) return;
    const int length = kv_length(a, b), shift = length - (int)rows.all, r0 = tile * a.tile_rows;
    const int r1 = r0 + a.tile_rows < rows.count * a.group ? r0 + a.tile_rows - 1 : rows.count * a.group - 1;
    const KvRange range = kv_range(a, length, a.causal ? shift + r0 / a.group : length - 1, a.causal ? shift + r1 / a.group : length - 1);
    const int per = kv_share(range.count, a.splits, a.tile_rows);
    int used = (range.count + per - 1) / per;
    used = used < 1 ? 1 : used;
    const float* ml = a.part_ml + slot * a.splits * 2;
#pragma unroll
    for (int i = 0; i < kKvMaxSplits / 64; ++i) {
        if (i % (kKvJoin / 64) != wave) continue;
        const int s = i * 64 + lane;
        const float m0 = s < used ? ml[2 * s] : -INFINITY, l0 = s < used ? ml[2 * s + 1] : 0.f;
        const float m1 = wave_max(m0), w = __builtin_amdgcn_exp2f(m0 - kv_finite(m1));
        weight[s] = l0 * w;                                      // relative to the largest of its 64 shares
        const float l1 = wave_sum(l0 * w);
        if (lane == 0) {
            box_m[i] = m1;
            box_l[i] = l1;
        }
    }
    __syncthreads();
    const float m = kv_finite(fmaxf(fmaxf(box_m[0], box_m[1]), fmaxf(box_m[2], box_m[3])));
    float f[4], l = 0.f;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        f[i] = __builtin_amdgcn_exp2f(box_m[i] - m);
        l += box_l[i] * f[i];
    }
    l = kv_inverse(l);
#pragma unroll
    for (int i = 0; i < 4; ++i) f[i] *= l;                       // shares sum to 1
    const int quads = a.D >> 2, lines = kKvJoin / quads;         // lanes of a row; rows (shares) read at once
    const int line = tid / quads, d = tid % quads * 4;
    kv_f32x4 acc = {0.f, 0.f, 0.f, 0.f};
    if (line < lines) {
        const float* p = a.part + slot * a.splits * a.D + d;
#pragma unroll 8
        for (int s = line; s < used; s += lines) {
            const float w = weight[s] * f[s >> 6];
            const kv_f32x4 v = *(const kv_f32x4*)(p + (int64_t)s * a.D);
#pragma unroll
            for (int e = 0; e < 4; ++e) acc[e] += v[e] * w;
        }
    }
    *(kv_f32x4*)(box + tid * 4) = acc;
    __syncthreads();
    T* o = (T*)a.o + (rows.first + tok) * a.o_tok + (h * a.group + row - tok * a.group) * a.o_head;
    for (int e = tid; e < a.D; e += kKvJoin) {
        float v = 0.f;
        for (int i = 0; i < lines && i < used; ++i) v += box[(i * quads + (e >> 2)) * 4 + (e & 3)];
        o[e] = from_f<T>(v);
    }
}

// How a call is cut.
//
// Tiles of 16 rows of a (sequence, key head), or of 128 or 64 where these are enough to fill the chip, which has room for 512 (for more
// than 128 features 256) workgroups of them: 128 rows from 512 workgroups on, 64 above 256, and only where a sequence has
// more than 16 rows on average (255 sequences of 2 queries behind 1000, `most` given as 510: 109 us in tiles of 16, 164 of 64).
// us with 8 key heads of 128 features and groups of 4 (16 / 64 / 128 rows): 2048 queries (512 tiles of 128) 150 / 92 / 75; up to 4 x 1024 behind 8000 keys 355 / 255 / 240; 4096
// queries of 8 ungrouped heads of 64 features 84 / 71 / 86; 512 queries (128 tiles) 30 / 24 / 28; 16 of up to 30 behind up to 1000 (128) 26 / 34 / 41; 100
// queries (32) 14 / 17 / 18.  float32 (three products): up to 2 x 2000 queries 202 / 218 / 163, up to 4 x 200 30 / 39 / 51.
//
// Then shares of the keys, until 512 workgroups have work.  Tiles of 16: no share less than 8 groups of 64 tokens.  us with 256 / 512 / 768 /
// 1024 workgroups, three states in turn: one token of 64 sequences of up to 4096 (8 key heads, 128 features) 57 / 57 / 62 / 62; of one sequence
// of 131071 37 / 39 / 42 / 42; of 16 windows of 2000 24 / 26 / 26 / 26; 4 queries of 16 sequences of up to 8000 48 / 45 / 51 / 49; 8 queries (two tiles) 87
// / 71 / 74 / 69.  Large tiles, whose partial results are many: only from 4 shares of 16 groups on
// (2048 queries as two shares 140 us, as one 71; 64 queries behind 60000 keys as 32 shares 104).
struct KvPlan {
    int tile_rows, tiles, splits;    // tiles of a sequence of `most` rows
    int64_t slots, grid;
};
static KvPlan kv_plan(int64_t all_rows, int sequences, int most, int64_t longest, int heads, int group, int dim, int window, int sinks,
                      int dtype) {
    KvPlan p;
    const int64_t rows = (int64_t)most * group;
    if (window > 0 && (int64_t)window + sinks + most < longest) longest = (int64_t)window + sinks + most;     // keys that a tile can see
    const int64_t groups = (longest + kKvGroup - 1) / kKvGroup;
    int64_t base;                    // workgroups of one share
    auto cut = [&](int tile_rows) {
        p.tile_rows = tile_rows;
        p.tiles = (int)((rows + tile_rows - 1) / tile_rows);
        int64_t tiles = (int64_t)sequences * p.tiles;
        // packed rows bound the tiles of all sequences together: whole ones, and one for what is left of each
        if (p.tiles > 1 && all_rows * group / tile_rows + sequences < tiles) tiles = all_rows * group / tile_rows + sequences;
        base = tiles * heads;
        p.slots = base * tile_rows;
        int64_t splits = base > 0 ? (512 + base - 1) / base : 1;
        if (splits > groups / kv_min_share(tile_rows)) splits = groups / kv_min_share(tile_rows);
        if (tile_rows > 16 && splits < 4) splits = 1;
        p.splits = splits < 1 ? 1 : splits > kKvMaxSplits ? kKvMaxSplits : (int)splits;
        return base * p.splits;
    };
    const bool large = rows > 64 && all_rows * group > 16 * (int64_t)sequences && !(dtype == VAMD_F32 && dim > 128);
    if (!large || (cut(128) < (dim > 128 ? 256 : 512) && cut(64) <= 256)) cut(16);
    p.grid = base * p.splits;
    return p;
}

template <typename T, int FMT> static int kv_launch_rows(const KvAttendArgs& a, int64_t grid, hipStream_t st) {
    const int C = (a.D + 63) / 64;
    const size_t lds = (size_t)(2 * 64 * C * 16 + 2 * 64 * 2) * 4;
#define KV_ROWS(C_)                                                                                                              \
    case C_:                                                                                                                     \
        if (a.tiles == 1) hipLaunchKernelGGL((kv_attend_rows_kernel<T, FMT, C_, true>), grid_of(grid), dim3(256), lds, st, a);      \
        else hipLaunchKernelGGL((kv_attend_rows_kernel<T, FMT, C_, false>), grid_of(grid), dim3(256), lds, st, a);        \
        break
    switch (C) {
        KV_ROWS(1);
        KV_ROWS(2);
        KV_ROWS(3);
        KV_ROWS(4);
    }
#undef KV_ROWS
    VAMD_LAUNCH_OK("kv_attend_rows");
    return 0;
}

template <typename T, int FMT, int DT, int KW> static int kv_launch_tile_of(const KvAttendArgs& a, int64_t grid, hipStream_t st) {
    constexpr int LDS = 2 * 2 * DT * 4 * 64 * 16;
    static_assert(KW == 1 || LDS >= 2 * (DT * 16 + 2) * 64 * 4, "the waves' results pass through the buffers");
    auto kernel = kv_attend_tile_kernel<T, FMT, DT, KW>;
    if (LDS > 64 * 1024) {
        const hipError_t e = hipFuncSetAttribute(reinterpret_cast<const void*>(kernel), hipFuncAttributeMaxDynamicSharedMemorySize, LDS);
        if (e != hipSuccess) return fail((int)e, "vamd_kv_attend: hipFuncSetAttribute failed: %s", hipGetErrorString(e));
    }
    hipLaunchKernelGGL(kernel, grid_of(grid), dim3(kKvTileThreads), LDS, st, a);
    VAMD_LAUNCH_OK("kv_attend_tile");
    return 0;
}
template <typename T, int FMT, int KW> static int kv_launch_tile(const KvAttendArgs& a, int64_t grid, hipStream_t st) {
    switch ((a.D + 31) / 32) {
        case 1: return kv_launch_tile_of<T, FMT, 1, KW>(a, grid, st);
        case 2: return kv_launch_tile_of<T, FMT, 2, KW>(a, grid, st);
        case 3: return kv_launch_tile_of<T, FMT, 3, KW>(a, grid, st);
        case 4: return kv_launch_tile_of<T, FMT, 4, KW>(a, grid, st);
    }
    if constexpr (sizeof(T) == 2) {
        switch ((a.D + 31) / 32) {
            case 5:
            case 6: return kv_launch_tile_of<T, FMT, 6, KW>(a, grid, st);
            default: return kv_launch_tile_of<T, FMT, 8, KW>(a, grid, st);
        }
    }
    return fail(VAMD_EUNSUPPORTED, "vamd_kv_attend: no kernel for %d features in float32", a.D);
}

// One wave per row, four or sixteen: so many that a lane reads about four shares.  32 rows of 256 shares: 12 us with four waves, 5.5 with
// sixteen; 512 rows of 4 shares (128 features): 18 us with sixteen waves, 5.5 with one.
template <typename T> static int kv_launch_join(const KvAttendArgs& a, hipStream_t st) {
    const unsigned grid = (unsigned)((int64_t)a.all_tiles * a.heads * kv_tile_fill(a.tiles, a.tile_rows, a.most, a.group));
    const int lanes = a.splits * (a.D / 4) / 4;
    if (lanes <= 64) hipLaunchKernelGGL((kv_join_kernel<T, 64>), dim3(grid), dim3(64), 0, st, a);
    else if (lanes <= 256) hipLaunchKernelGGL((kv_join_kernel<T, 256>), dim3(grid), dim3(256), 0, st, a);
    else hipLaunchKernelGGL((kv_join_kernel<T, 1024>), dim3(grid), dim3(1024), 0, st, a);
    VAMD_LAUNCH_OK("kv_join");
    return 0;
}

}  // namespace vamd

using namespace vamd;

extern "C" size_t vamd_kv_attend_workspace(int64_t rows, int sequences, int most, int64_t longest, int heads, int group, int dim, int window, int sinks,
                                           int dtype) {
    if (rows <= 0 || sequences <= 0 || most <= 0 || heads <= 0 || group <= 0 || dim <= 0) return 0;
    const KvPlan p = kv_plan(rows, sequences, most, longest, heads, group, dim, window, sinks, dtype);
    return p.splits > 1 ? (size_t)p.slots * p.splits * (dim + 2) * sizeof(float) : 0;
}

extern "C" int vamd_kv_attend_tile(int64_t rows, int sequences, int most, int64_t longest, int heads, int group, int dim, int window, int sinks,
                                   int dtype) {
    if (rows <= 0 || sequences <= 0 || most <= 0 || heads <= 0 || group <= 0 || dim <= 0) return 0;
    return kv_plan(rows, sequences, most, longest, heads, group, dim, window, sinks, dtype).tile_rows;
}

extern "C" int vamd_kv_attend(const void* q, int64_t q_token, int64_t q_head, const void* codes_k, const void* codes_v,
                              const float* scales_k, const float* scales_v, const int32_t* table, int64_t table_stride,
                              const int32_t* lengths, const int32_t* offsets, int64_t rows, int sequences, int most, int64_t longest,
                              int heads, int group, int dim, int block, int width, int blocks, int format, float scale, int causal,
                              int window, int sinks, void* o, int64_t o_token, int64_t o_head, void* workspace, size_t workspace_bytes,
                              int dtype, void* stream) {
    VAMD_REQUIRE(sequences > 0 && rows >= 0 && most >= 0 && heads > 0 && heads <= 65536 && group > 0 && group <= 65536 && width > 0 &&
                 blocks > 0 && table_stride >= 0, "vamd_kv_attend: bad extents (%d sequences, %lld rows, most %d, %d key heads x %d, %d "
                 "blocks a sequence of %d)", sequences, (long long)rows, most, heads, group, width, blocks);
    VAMD_REQUIRE(dim >= 16 && dim <= 256 && dim % 16 == 0, "vamd_kv_attend: dim %d (a multiple of 16, 16 to 256)", dim);
    VAMD_REQUIRE(block == 64 || block == 128 || block == 256, "vamd_kv_attend: block %d (64, 128 or 256 tokens)", block);
    VAMD_REQUIRE(format == VAMD_KV_E4M3 || format == VAMD_KV_INT8, "vamd_kv_attend: bad format %d", format);
    VAMD_REQUIRE(dtype == VAMD_F32 || dtype == VAMD_BF16, "vamd_kv_attend: bad dtype %d", dtype);
    VAMD_REQUIRE(window >= 0 && sinks >= 0 && (causal || window == 0), "vamd_kv_attend: window %d, sinks %d (not negative; a window "
                 "needs causal queries)", window, sinks);
    VAMD_REQUIRE((int64_t)width * block <= 0x7fffffc0, "vamd_kv_attend: %d blocks of %d tokens are too many for a sequence", width, block);
    // (64 sequences' tiles are counted at once)
    VAMD_REQUIRE((int64_t)most * group <= 1 << 28 && rows <= 0x7fffffff, "vamd_kv_attend: %d of %lld rows of %d heads are too many for a sequence",
                 most, (long long)rows, group);
    VAMD_REQUIRE(offsets || rows == (int64_t)sequences * most, "vamd_kv_attend: %lld rows are not %d for each of %d sequences",
                 (long long)rows, most, sequences);
    if (rows == 0 || most == 0) return 0;
    VAMD_REQUIRE(q && o && codes_k && codes_v && scales_k && scales_v && table && lengths, "vamd_kv_attend: NULL tensor");
    const int size = dtype == VAMD_BF16 ? 2 : 4;
    VAMD_REQUIRE((uintptr_t)codes_k % 16 == 0 && (uintptr_t)codes_v % 16 == 0 && (uintptr_t)scales_k % 4 == 0 && (uintptr_t)scales_v % 4 == 0 &&
                 (uintptr_t)table % 4 == 0 && (uintptr_t)lengths % 4 == 0 && (uintptr_t)offsets % 4 == 0 && (uintptr_t)q % size == 0 &&
                 (uintptr_t)o % size == 0, "vamd_kv_attend: misaligned tensor");
    const KvPlan plan = kv_plan(rows, sequences, most, longest, heads, group, dim, window, sinks, dtype);
    const size_t need = vamd_kv_attend_workspace(rows, sequences, most, longest, heads, group, dim, window, sinks, dtype);
    VAMD_REQUIRE(need == 0 || (workspace && (uintptr_t)workspace % 16 == 0 && workspace_bytes >= need),
                 "vamd_kv_attend: workspace of %zu bytes, %zu needed (16-byte aligned)", workspace_bytes, need);
    const int64_t grid = plan.grid;
    VAMD_REQUIRE(grid <= kGridMost, "vamd_kv_attend: %d sequences of up to %d rows are too many for one call",
                 sequences, most);
    KvAttendArgs a = {};
    a.q = q;
    a.o = o;
    a.q_tok = q_token;
    a.q_head = q_head;
    a.o_tok = o_token;
    a.o_head = o_head;
    a.codes[0] = (const uint8_t*)codes_k;
    a.codes[1] = (const uint8_t*)codes_v;
    a.scales[0] = scales_k;
    a.scales[1] = scales_v;
    a.table = table;
    a.table_stride = table_stride;
    a.lengths = lengths;
    a.offsets = offsets;
    a.rows = rows;
    a.part = (float*)workspace;
    a.part_ml = a.part + (size_t)plan.slots * plan.splits * dim;
    a.scale2 = scale * 1.44269504088896340736f;
    a.sequences = sequences;
    a.most = most;
    a.heads = heads;
    a.group = group;
    a.D = dim;
    a.block_shift = block == 64 ? 6 : block == 128 ? 7 : 8;
    a.width = width;
    a.blocks = blocks;
    a.window = window;
    a.sinks = sinks;
    a.causal = causal;
    a.tiles = plan.tiles;
    a.all_tiles = (int)(plan.grid / plan.splits / heads);
    a.tile_rows = plan.tile_rows;
    a.splits = plan.splits;
    const int n = 16 / size;
    a.q_aligned = (uintptr_t)q % 16 == 0 && q_token % n == 0 && q_head % n == 0;
    a.o_aligned = (uintptr_t)o % (4 * size) == 0 && o_token % 4 == 0 && o_head % 4 == 0;
    hipStream_t st = as_stream(stream);
    auto launch = [&](auto t, auto f) {
        using T = decltype(t);
        constexpr int FMT = decltype(f)::value;
        return plan.tile_rows == 16   ? kv_launch_rows<T, FMT>(a, grid, st)
               : plan.tile_rows == 64 ? kv_launch_tile<T, FMT, 2>(a, grid, st)
                                      : kv_launch_tile<T, FMT, 1>(a, grid, st);
    };
    const std::integral_constant<int, VAMD_KV_E4M3> e4m3;
    const std::integral_constant<int, VAMD_KV_INT8> int8;
    int rc;
    if (dtype == VAMD_BF16) rc = format == VAMD_KV_E4M3 ? launch(bf16_t(), e4m3) : launch(bf16_t(), int8);
    else rc = format == VAMD_KV_E4M3 ? launch(float(), e4m3) : launch(float(), int8);
    if (rc || plan.splits == 1) return rc;
    return dtype == VAMD_BF16 ? kv_launch_join<bf16_t>(a, st) : kv_launch_join<float>(a, st);
}
