// Rotary positions: pairs (x1, x2) of a head's first `turned` features are turned by the angle position * frequency,
//
//     y1 = a (x1 cos - x2 sin),  y2 = a (x2 cos + x1 sin)        (a: amplitude; `inverse`: sin -> -sin, which is the gradient)
//
// with the pairs (i, i + turned / 2) ("half") or (2i, 2i + 1) ("interleaved"); the features behind them are copied.
//
// Angles.  A float32 angle is wrong by 0.06 at position 10^6.  Frequencies therefore come in turns, as 64-bit fixed-point
// fractions, and position * frequency is a 64-bit integer product whose overflow drops whole turns: the fraction of a turn is
// exact to 2^-64 times the position at any distance, without a division.  The nearest quarter turn is split off the top two
// bits, the rest (|x| <= pi/4) goes into the Taylor polynomials of sine (to x^9) and cosine (to x^10): 2e-9 at the border.
//
// Memory bound: every element is read and written once, in pieces of 16 bytes where the layout allows it.  One lane owns
// 2 V features (V pairs' halves, or V whole pairs) of one token and walks over `per` heads of both tensors, so that the
// angles of a token are computed once for `per` heads; neighbouring lanes own neighbouring pieces of a row.  16383 tokens of 32 + 8
// heads of 128 features in bf16: 65 us, 5.1 TB/s (a large copy: 5.2); 4099 tokens of 16 + 16 heads of 96 in float32: 29 us, 3.5 (21 us where
// the inputs are still in the caches).
#include "common.h"

namespace vamd {

struct RotaryRows {
    const void* x;
    void* y;
    int64_t xb, xt, xh, yb, yt, yh;      // strides of a batch, a token and a head, in elements
    int heads;
};

struct RotaryArgs {
    RotaryRows t[2];
    const void* positions;
    const uint64_t* frequencies;
    float amplitude;
    int wide, turned, dim, interleaved, inverse;
    int chunks, per, slots;      // lanes a row; heads a lane walks over; lanes over the heads
    int64_t batch, tokens;       // tokens of a batch
};

// cos and sin of `phase` / 2^64 turns
__device__ __forceinline__ void rotary_angle(uint64_t phase, float& c, float& s) {
    const uint64_t shifted = phase + (1ull << 61);
    const uint32_t quarter = (uint32_t)(shifted >> 62);
    const int64_t rest = (int64_t)(phase - ((uint64_t)quarter << 62));        // -2^61 .. 2^61: an eighth of a turn
    const float f = fmaf((float)(uint32_t)rest, 0x1p-64f, (float)(int32_t)(rest >> 32) * 0x1p-32f);
    const float x = f * 6.28318530717958647692f, z = x * x;
    const float sp = fmaf(z, fmaf(z, fmaf(z, 1.f / 362880.f, -1.f / 5040.f), 1.f / 120.f), -1.f / 6.f);
    const float sn = fmaf(x * z, sp, x);
    const float cp = fmaf(z, fmaf(z, fmaf(z, -1.f / 3628800.f, 1.f / 40320.f), -1.f / 720.f), 1.f / 24.f);
    const float cs = fmaf(z, fmaf(z, cp, -0.5f), 1.f);
    const float a = quarter & 1 ? sn : cs, b = quarter & 1 ? cs : sn;
    c = (quarter == 1 || quarter == 2) ? -a : a;
    s = quarter >= 2 ? -b : b;
}

template <typename T, int V> struct alignas(sizeof(T) * V) RotaryPiece { T v[V]; };

template <typename T, int V>
__global__ void __launch_bounds__(256) rotary_kernel(const RotaryArgs a) {
    typedef RotaryPiece<T, V> Piece;
    const int64_t id = (int64_t)block_number() * 256 + threadIdx.x;
    const int64_t rest = id / a.chunks;
    const int chunk = (int)(id - rest * a.chunks);
    const int64_t at = rest / a.slots;
    const int slot = (int)(rest - at * a.slots);
    if (at >= a.batch * a.tokens) return;
    const int64_t b = at / a.tokens, token = at - b * a.tokens;
    const int half = a.turned >> 1, first = slot * a.per;
    const int heads = a.t[0].heads + a.t[1].heads;
    const int last = first + a.per < heads ? first + a.per : heads;
    const int d = chunk * (a.interleaved ? 2 * V : V);
    if (d < (a.interleaved ? a.turned : half)) {
        const int p0 = a.interleaved ? d >> 1 : d;               // the lane's first pair
        const uint64_t pos = (uint64_t)(a.wide ? ((const int64_t*)a.positions)[at] : (int64_t)((const int32_t*)a.positions)[at]);
        float c[V], s[V];
#pragma unroll
        for (int i = 0; i < V; ++i) {
            rotary_angle(pos * a.frequencies[p0 + i], c[i], s[i]);
            c[i] *= a.amplitude;
            s[i] *= a.inverse ? -a.amplitude : a.amplitude;
        }
        const int step = a.interleaved ? V : half;
#pragma unroll 4
        for (int h = first; h < last; ++h) {
            const RotaryRows& t = h < a.t[0].heads ? a.t[0] : a.t[1];
            const int hh = h < a.t[0].heads ? h : h - a.t[0].heads;
            const T* x = (const T*)t.x + b * t.xb + token * t.xt + hh * t.xh + d;
            T* y = (T*)t.y + b * t.yb + token * t.yt + hh * t.yh + d;
            Piece u = *(const Piece*)x, w = *(const Piece*)(x + step);
            if (a.interleaved) {
                // pairs lie side by side: the first V / 2 in u, the others in w (V = 1: the pair is u, w)
                if (V == 1) {
                    const float x1 = to_f(u.v[0]), x2 = to_f(w.v[0]);
                    u.v[0] = from_f<T>(fmaf(x1, c[0], -(x2 * s[0])));
                    w.v[0] = from_f<T>(fmaf(x2, c[0], x1 * s[0]));
                } else {
#pragma unroll
                    for (int i = 0; i < V / 2; ++i) {
                        const float x1 = to_f(u.v[2 * i]), x2 = to_f(u.v[2 * i + 1]);
                        u.v[2 * i] = from_f<T>(fmaf(x1, c[i], -(x2 * s[i])));
                        u.v[2 * i + 1] = from_f<T>(fmaf(x2, c[i], x1 * s[i]));
                        const float x3 = to_f(w.v[2 * i]), x4 = to_f(w.v[2 * i + 1]);
                        w.v[2 * i] = from_f<T>(fmaf(x3, c[V / 2 + i], -(x4 * s[V / 2 + i])));
                        w.v[2 * i + 1] = from_f<T>(fmaf(x4, c[V / 2 + i], x3 * s[V / 2 + i]));
                    }
                }
            } else {
#pragma unroll
                for (int i = 0; i < V; ++i) {
                    const float x1 = to_f(u.v[i]), x2 = to_f(w.v[i]);
                    u.v[i] = from_f<T>(fmaf(x1, c[i], -(x2 * s[i])));
                    w.v[i] = from_f<T>(fmaf(x2, c[i], x1 * s[i]));
                }
            }
            *(Piece*)y = u;
            *(Piece*)(y + step) = w;
        }
    } else {
        // features that are not turned: 2 V a lane, the last lane of a row maybe V
        const int d0 = a.turned + (chunk - (half + V - 1) / V) * 2 * V;
        for (int h = first; h < last; ++h) {
            const RotaryRows& t = h < a.t[0].heads ? a.t[0] : a.t[1];
            const int hh = h < a.t[0].heads ? h : h - a.t[0].heads;
            const T* x = (const T*)t.x + b * t.xb + token * t.xt + hh * t.xh;
            T* y = (T*)t.y + b * t.yb + token * t.yt + hh * t.yh;
            if (x == y) continue;                                // in place: nothing to copy
#pragma unroll
            for (int i = 0; i < 2; ++i)
                if (d0 + i * V < a.dim) *(Piece*)(y + d0 + i * V) = *(const Piece*)(x + d0 + i * V);
        }
    }
}

// What a piece of V elements needs: it divides the halves and the rest of a row, and every row starts on its boundary.
static bool rotary_fits(const RotaryArgs& a, int V, int size) {
    if ((a.turned / 2) % V || (a.dim - a.turned) % V) return false;
    for (const RotaryRows& t : a.t) {
        if (!t.heads) continue;
        if (t.xb % V || t.yb % V || t.xt % V || t.xh % V || t.yt % V || t.yh % V || (uintptr_t)t.x % (V * size) || (uintptr_t)t.y % (V * size)) return false;
    }
    return true;
}

template <typename T> static int rotary_launch(RotaryArgs& a, hipStream_t st) {
    int V = 16 / sizeof(T);
    while (V > 1 && !rotary_fits(a, V, sizeof(T))) V >>= 1;
    a.chunks = (a.turned / 2 + V - 1) / V + (a.dim - a.turned + 2 * V - 1) / (2 * V);
    const int heads = a.t[0].heads + a.t[1].heads;
    // A lane walks over 8 heads once that still leaves 16 waves to each of the 256 CUs, over fewer before that.
    a.per = 8;
    const double lanes = (double)(a.batch * a.tokens) * a.chunks;      // (of one head; the product with the heads' may pass 64 bits)
    while (a.per > 1 && lanes * ((heads + a.per - 1) / a.per) < 256 * 16 * 64) a.per >>= 1;
    a.slots = (heads + a.per - 1) / a.per;
    VAMD_REQUIRE(lanes * a.slots <= 256.0 * kGridMost, "vamd_rotary: %lld tokens of %d heads are too many for one call",
                 (long long)(a.batch * a.tokens), heads);
    const int64_t blocks = (a.batch * a.tokens * a.chunks * a.slots + 255) / 256;
    const dim3 grid = grid_of(blocks);
    if (V == 8) {
        if constexpr (sizeof(T) == 2) hipLaunchKernelGGL((rotary_kernel<T, 8>), grid, dim3(256), 0, st, a);
    } else if (V == 4) hipLaunchKernelGGL((rotary_kernel<T, 4>), grid, dim3(256), 0, st, a);
    else if (V == 2) hipLaunchKernelGGL((rotary_kernel<T, 2>), grid, dim3(256), 0, st, a);
    else hipLaunchKernelGGL((rotary_kernel<T, 1>), grid, dim3(256), 0, st, a);
    VAMD_LAUNCH_OK("rotary");
    return 0;
}

}  // namespace vamd

using namespace vamd;

extern "C" int vamd_rotary(const void* positions, int wide, const uint64_t* frequencies, float amplitude, int64_t batch, int64_t tokens,
                           int dim, int turned, int interleaved, int inverse, const void* q, void* yq, int q_heads, int64_t q_batch,
                           int64_t q_token, int64_t q_head, int64_t yq_batch, int64_t yq_token, int64_t yq_head, const void* k, void* yk,
                           int k_heads, int64_t k_batch, int64_t k_token, int64_t k_head, int64_t yk_batch, int64_t yk_token,
                           int64_t yk_head, int dtype, void* stream) {
    VAMD_REQUIRE(batch >= 0 && tokens >= 0 && batch <= 0x7fffffff && tokens <= 0x7fffffff && dim >= 2 && dim <= 65536,
                 "vamd_rotary: bad extents (%lld x %lld tokens, dim %d)", (long long)batch, (long long)tokens, dim);
    VAMD_REQUIRE(turned >= 2 && turned <= dim && turned % 2 == 0, "vamd_rotary: %d of %d features cannot be turned (an even number, 2 "
                 "to the head's size)", turned, dim);
    VAMD_REQUIRE(dtype == VAMD_F32 || dtype == VAMD_BF16, "vamd_rotary: bad dtype %d", dtype);
    VAMD_REQUIRE(q_heads >= 0 && k_heads >= 0 && q_heads <= 65536 && k_heads <= 65536, "vamd_rotary: bad number of heads (%d, %d)", q_heads, k_heads);
    if (batch == 0 || tokens == 0 || q_heads + k_heads == 0) return 0;
    VAMD_REQUIRE(positions && frequencies && (q_heads == 0 || (q && yq)) && (k_heads == 0 || (k && yk)), "vamd_rotary: NULL tensor");
    const int size = dtype == VAMD_BF16 ? 2 : 4;
    VAMD_REQUIRE((uintptr_t)positions % (wide ? 8 : 4) == 0 && (uintptr_t)frequencies % 8 == 0 && (uintptr_t)q % size == 0 &&
                 (uintptr_t)yq % size == 0 && (uintptr_t)k % size == 0 && (uintptr_t)yk % size == 0, "vamd_rotary: misaligned tensor");
    RotaryArgs a = {};
    a.t[0] = RotaryRows{q, yq, q_batch, q_token, q_head, yq_batch, yq_token, yq_head, q_heads};
    a.t[1] = RotaryRows{k, yk, k_batch, k_token, k_head, yk_batch, yk_token, yk_head, k_heads};
    a.positions = positions;
    a.frequencies = frequencies;
    a.amplitude = amplitude;
    a.wide = wide;
    a.turned = turned;
    a.dim = dim;
    a.interleaved = interleaved;
    a.inverse = inverse;
    a.batch = batch;
    a.tokens = tokens;
    return dtype == VAMD_BF16 ? rotary_launch<bf16_t>(a, as_stream(stream)) : rotary_launch<float>(a, as_stream(stream));
}
