// What the kernels that turn heads by their positions share (rotary.hip, head_norm.hip, paged_int8.hip): angles, turns, a lane's place in a head.
#pragma once
#include "paged.h"

#define ROW_WAVES 4  // waves, each of a token and a slice of heads, per workgroup
#define PASSES 4     // heads per lane
#define MAX_PAIRS 128
#define MAX_ROWS ((1L << 26) - 64)  // tokens of a call: a grid has fewer than 2^32 threads

// Cosine and sine of a turn's fraction: n f - rint(4 n f) / 4 = y / 4, |y| <= 1/2, then the series at y pi / 2 (at most pi / 4:
// the first terms left out are below 2e-9 and 1.2e-10).
__device__ __forceinline__ f2 cos_sin(double position, double turns) {
    const double quarters = 4.0 * (position * turns), whole = rint(quarters);
    const float y = (float)(quarters - whole), z = y * y;
    const int quadrant = (int)(whole - 4.0 * rint(whole * 0.25)) & 3;
    float s = 1.60441184787359821e-4f;
    s = __builtin_fmaf(s, z, -4.68175413531868810e-3f);
    s = __builtin_fmaf(s, z, 7.96926262461670451e-2f);
    s = __builtin_fmaf(s, z, -6.45964097506246254e-1f);
    s = __builtin_fmaf(s, z, 1.57079632679489662f) * y;
    float c = -2.52020423730606055e-5f;
    c = __builtin_fmaf(c, z, 9.19260274839426580e-4f);
    c = __builtin_fmaf(c, z, -2.08634807633529609e-2f);
    c = __builtin_fmaf(c, z, 2.53669507901048014e-1f);
    c = __builtin_fmaf(c, z, -1.23370055013616983f);
    c = __builtin_fmaf(c, z, 1.f);
    const float cos = quadrant & 1 ? s : c, sin = quadrant & 1 ? c : s;
    return (f2){quadrant == 1 || quadrant == 2 ? -cos : cos, quadrant >= 2 ? -sin : sin};
}

struct RotaryArgs {
    const double* turns;  // R / 2 frequencies, turns per position
    int D, R, interleaved;
    float factor, sign;  // sign -1: by the negative angle
};

// The wave's token's cosines and sines, pair i at cs[i]; the lanes' angles of position n.
__device__ __forceinline__ void make_angles(const RotaryArgs& r, double f0, double f1, double n, f2* cs, int lane) {
    const int pairs = r.R / 2;
    if (lane < pairs) {
        const f2 v = cos_sin(n, f0);
        cs[lane] = (f2){v[0] * r.factor, v[1] * r.factor * r.sign};
    }
    if (lane + 64 < pairs) {
        const f2 v = cos_sin(n, f1);
        cs[lane + 64] = (f2){v[0] * r.factor, v[1] * r.factor * r.sign};
    }
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
}

// Turns a lane's eight pairs, held as two vectors: half layout (a[i], b[i]), interleaved (a[2 i], a[2 i + 1]) and so on into b.
__device__ __forceinline__ void turn(f8& a, f8& b, const f8& c, const f8& s, bool interleaved) {
    f8 x = a, y = b;
    if (interleaved) {
        x = __builtin_shufflevector(a, b, 0, 2, 4, 6, 8, 10, 12, 14);
        y = __builtin_shufflevector(a, b, 1, 3, 5, 7, 9, 11, 13, 15);
    }
    f8 u, v;
#pragma unroll
    for (int i = 0; i < 8; i++) {
        u[i] = __builtin_fmaf(x[i], c[i], -(y[i] * s[i]));
        v[i] = __builtin_fmaf(x[i], s[i], y[i] * c[i]);
    }
    a = interleaved ? __builtin_shufflevector(u, v, 0, 8, 1, 9, 2, 10, 3, 11) : u;
    b = interleaved ? __builtin_shufflevector(u, v, 4, 12, 5, 13, 6, 14, 7, 15) : v;
}

// A lane's place in a head: D / 16 lanes hold a head, 64 / (D / 16) heads go to a pass. Lanes past whole heads have no work.
struct Place {
    int head, heads;  // first head within the slice; heads per pass
    int at, to;       // offsets of the two vectors
    int pair;         // first pair, or -1 where the values are copied
};
__device__ __forceinline__ Place place(const RotaryArgs& r, int lane) {
    const int per = r.D / 16, u = lane % per;
    Place p;
    p.heads = 64 / per;
    p.head = lane / per;
    const bool turned = u < r.R / 16;
    p.at = turned && !r.interleaved ? 8 * u : 16 * u;
    p.to = turned && !r.interleaved ? 8 * u + r.R / 2 : 16 * u + 8;
    p.pair = turned ? 8 * u : -1;
    return p;
}
__device__ __forceinline__ void angles_of(const Place& p, const f2* cs, f8& c, f8& s) {
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const f4 v = ((const f4*)(cs + (p.pair < 0 ? 0 : p.pair)))[i];
        c[2 * i] = v[0];
        s[2 * i] = v[1];
        c[2 * i + 1] = v[2];
        s[2 * i + 1] = v[3];
    }
}

// The number of starts[1 .. B] at or below t: the sequence of row t (B: behind the last). 64 entries a step, one per lane.
__device__ __forceinline__ int sequence_of(const int* starts, int B, int t, int lane) {
    int at = 0, n = B;  // the answer is at .. at + n
    while (n > 64) {
        const int step = (n + 63) >> 6, i = (lane + 1) * step;
        const bool below = i <= n && starts[at + i] <= t;
        const int c = __popcll(__ballot(below));
        at += c * step;
        n = min(step - 1, n - c * step);
    }
    const bool below = lane < n && starts[at + 1 + lane] <= t;
    return at + __popcll(__ballot(below));
}

static bool rotary_ok(const double* turns, long D, long R) {
    return D > 0 && D % 16 == 0 && D <= 2 * MAX_PAIRS && R >= 0 && R % 16 == 0 && R <= D && (R == 0 || turns);
}

// ------------------------------------------------------------------------------------------------ norms of heads

// Eight weights of a head's norm as fp32, from any of the three types.
__device__ __forceinline__ f8 weights8(const void* w, int type, int at) {
    return type == RDA_FP16 ? load8((const half_t*)w + at) : type == RDA_BF16 ? load8((const bf16_t*)w + at) : load8((const float*)w + at);
}
// The sum over the `per` lanes that hold a head (lane / per is the head's place): by lane swaps where per is a power of two.
__device__ __forceinline__ float head_sum(float x, int per, int lane) {
    if ((per & (per - 1)) == 0) {
        if (per >= 2) x += dpp<0xB1>(x);
        if (per >= 4) x += dpp<0x4E>(x);
        if (per >= 8) x += dpp<0x141>(x);
        if (per >= 16) x += dpp<0x140>(x);
        return x;
    }
    const int base = lane - lane % per;
    float s = 0.f;
    for (int i = 0; i < per; i++) s += __shfl(x, base + i);
    return s;
}
__device__ __forceinline__ float dot16(const f8& a, const f8& b, const f8& c, const f8& d) {
    float s = 0.f;
#pragma unroll
    for (int i = 0; i < 8; i++) s = __builtin_fmaf(a[i], b[i], s);
#pragma unroll
    for (int i = 0; i < 8; i++) s = __builtin_fmaf(c[i], d[i], s);
    return s;
}
// 1 / sqrt(mean of the head's squares + eps), in 32 bits.
__device__ __forceinline__ float inverse_rms(const f8& lo, const f8& hi, int D, float eps, int per, int lane) {
    return 1.f / sqrtf(head_sum(dot16(lo, lo, hi, hi), per, lane) * (1.f / (float)D) + eps);
}
