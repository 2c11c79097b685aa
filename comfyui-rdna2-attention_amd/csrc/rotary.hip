// Rotary positions, alone and on the way into a paged key/value cache.
//
// A head's first R values are R / 2 pairs -- (i, i + R / 2) in the half layout, (2 i, 2 i + 1) in the interleaved one -- and pair i
// of a token at position n turns by the angle 2 pi n f_i, f_i in turns per position: (a, b) -> (a c - b s, a s + b c), c and s the
// angle's cosine and sine times a constant factor. Values past R are copied.
//
// n f_i is a product in 64 bits and loses its whole turns there: in 32 bits an angle near position 10^6 would be off by 0.06
// radians. What is left, at most half a quarter turn, goes to 32 bits and through the Taylor series of sine and cosine.
//
// Both kernels move every value once and do little else, so memory bounds them. A wave takes one token and up to PASSES x 64 / (D / 16)
// of its heads: its lanes make the token's angles once, one or two each, and share them through LDS (a lane that made the eight
// angles of its own pairs would spend ~300 instructions for each 32 bytes it moves). A lane then holds two vectors of eight values:
// the two halves of eight pairs. All of its loads go out before the angles are made.
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

struct RotateArgs {
    RotaryArgs r;
    const void* x;
    void* y;
    const void* positions;
    int wide;  // positions are 64-bit
    int L, H;
    long tokens, sxb, sxl, sxh, syb, syl, syh;
};

// Each value is read and written once: 4096 x 32 x 128 bf16 12.2 us, 5.5 TB/s, 9293 x 24 x 128 fp16 interleaved 21.6 us, 5.3 TB/s, where a
// copy of 1 GiB moves 5.2 TB/s. One token of 32 heads: 2.8 us, the latency of a launch and of two loads one after the other.
template <class X>
__global__ __launch_bounds__(ROW_WAVES * 64) void rotate_kernel(RotateArgs p) {
    __shared__ __attribute__((aligned(16))) f2 cs_all[ROW_WAVES][MAX_PAIRS];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const long token = (long)blockIdx.x * ROW_WAVES + wave;
    if (token >= p.tokens) return;
    f2* cs = cs_all[wave];
    const Place pl = place(p.r, lane);
    const long b = token / p.L, l = token % p.L;
    const double n = p.wide ? (double)((const long*)p.positions)[token] : (double)((const int*)p.positions)[token];
    const int pairs = p.r.R / 2;
    const double f0 = p.r.turns[min(lane, pairs - 1)], f1 = p.r.turns[min(lane + 64, pairs - 1)];
    const X* x = (const X*)p.x + b * p.sxb + l * p.sxl;
    X* y = (X*)p.y + b * p.syb + l * p.syl;
    const int first = blockIdx.y * pl.heads * PASSES + pl.head, end = pl.head < pl.heads ? p.H : 0;
    f8 lo[PASSES], hi[PASSES];
#pragma unroll
    for (int i = 0; i < PASSES; i++) {
        const int h = first + i * pl.heads;
        const X* src = x + (long)(h < end ? h : 0) * p.sxh;
        lo[i] = load8(src + pl.at);
        hi[i] = load8(src + pl.to);
    }
    make_angles(p.r, f0, f1, n, cs, lane);
    f8 c, s;
    angles_of(pl, cs, c, s);
#pragma unroll
    for (int i = 0; i < PASSES; i++) {
        const int h = first + i * pl.heads;
        if (pl.pair >= 0) turn(lo[i], hi[i], c, s, p.r.interleaved);
        if (h < end) {
            store8(y + (long)h * p.syh + pl.at, lo[i]);
            store8(y + (long)h * p.syh + pl.to, hi[i]);
        }
    }
}

struct AppendArgs {
    RotaryArgs r;
    const void *q, *k, *v;
    void *qo, *kp, *vp;
    const int *table, *starts, *lengths;
    int T, H, Hkv, B, N, P;
    Div S;
    long pitch, sqt, sqh, skt, skh, svt, svh, sot, soh, kpp, kpr, kph, vpp, vpr, vph;
};

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

// One step's keys and values to their pages, k rotated by its position on the way, and q rotated: a token's H query heads, Hkv key
// heads and Hkv value heads in this order are its heads. Rows of no sequence, positions outside the table and pages outside the
// cache write nothing (rows of a sequence still have their q rotated). All rows are loaded before the search for the token's sequence and its
// table entry, which are two to three loads one after the other. 16384 tokens of 32 + 2 x 8 heads of 128 fp16: 77 us, 5.2 TB/s; 64 single
// tokens: 4.8 us, those latencies; fp32 rows into bf16 pages (130 MB) 23 us, 5.6 TB/s.
template <class X, class C>
__global__ __launch_bounds__(ROW_WAVES * 64) void append_kernel(AppendArgs p) {
    __shared__ __attribute__((aligned(16))) f2 cs_all[ROW_WAVES][MAX_PAIRS];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int token = blockIdx.x * ROW_WAVES + wave;
    if (token >= p.T) return;
    f2* cs = cs_all[wave];
    const Place pl = place(p.r, lane);
    const int heads = p.H + 2 * p.Hkv;
    const int first = blockIdx.y * pl.heads * PASSES + pl.head, end = pl.head < pl.heads ? heads : 0;
    f8 lo[PASSES], hi[PASSES];
#pragma unroll
    for (int i = 0; i < PASSES; i++) {
        const int h = min(first + i * pl.heads, heads - 1), hk = h - p.H, hv = hk - p.Hkv;
        const X* src = hk < 0   ? (const X*)p.q + token * p.sqt + h * p.sqh
                       : hv < 0 ? (const X*)p.k + token * p.skt + hk * p.skh
                                : (const X*)p.v + token * p.svt + hv * p.svh;
        lo[i] = load8(src + pl.at);
        hi[i] = load8(src + pl.to);
    }
    const int pairs = p.r.R / 2;
    double f0 = 0, f1 = 0;
    if (pairs) {
        f0 = p.r.turns[min(lane, pairs - 1)];
        f1 = p.r.turns[min(lane + 64, pairs - 1)];
    }
    const int b = __builtin_amdgcn_readfirstlane(sequence_of(p.starts, p.B, token, lane));
    if (b >= p.B || token < p.starts[b]) return;
    const long n = (long)p.lengths[b] - p.starts[b + 1] + token;  // below 2^31 in size
    const int block = n >= 0 ? div_by((int)n, p.S) : p.N, row = (int)n - block * (int)p.S.d;
    int page = -1;
    if (block < p.N) page = p.table[b * p.pitch + block];
    make_angles(p.r, f0, f1, (double)n, cs, lane);
    f8 c, s;
    angles_of(pl, cs, c, s);
#pragma unroll
    for (int i = 0; i < PASSES; i++) {
        const int h = first + i * pl.heads, hk = h - p.H, hv = hk - p.Hkv;
        if (h >= end) continue;
        if (pl.pair >= 0 && hv < 0) turn(lo[i], hi[i], c, s, p.r.interleaved);
        if (hk >= 0 && (page < 0 || page >= p.P)) continue;
        C* dst = hk < 0   ? (C*)p.qo + token * p.sot + h * p.soh
                 : hv < 0 ? (C*)p.kp + page * p.kpp + row * p.kpr + hk * p.kph
                          : (C*)p.vp + page * p.vpp + row * p.vpr + hv * p.vph;
        store8(dst + pl.at, lo[i]);
        store8(dst + pl.to, hi[i]);
    }
}

// Values are read and written in vectors of eight: 16-byte aligned bases and strides.
static bool vector_rows(const void* p, const long* strides, int n, int type) {
    const long m = type == RDA_FP32 ? 4 : 8;
    for (int i = 0; i < n; i++)
        if (strides[i] % m) return false;
    return ((uintptr_t)p & 15) == 0;
}
static bool rotary_ok(const double* turns, long D, long R) {
    return D > 0 && D % 16 == 0 && D <= 2 * MAX_PAIRS && R >= 0 && R % 16 == 0 && R <= D && (R == 0 || turns);
}

extern "C" {

int rda_rotate_positions(const void* x, void* y, const void* positions, int wide, const double* turns, float factor, int flags, int type, const long* dims,
                         void* stream) {
    const long B = dims[0], L = dims[1], H = dims[2], D = dims[3], R = dims[4];
    if (B <= 0 || L <= 0 || H <= 0 || H > 65535 || !rotary_ok(turns, D, R) || R == 0) return RDA_ERR_INVALID;
    const long groups = (B * L + ROW_WAVES - 1) / ROW_WAVES, slice = 64 / (D / 16) * PASSES;
    if (B > MAX_ROWS || L > MAX_ROWS || B * L > MAX_ROWS || type < RDA_FP16 || type > RDA_FP32 || !vector_rows(x, dims + 5, 3, type) || !vector_rows(y, dims + 8, 3, type))
        return RDA_ERR_INVALID;
    const RotateArgs a = {{turns, (int)D, (int)R, flags & 1, factor, flags & 2 ? -1.f : 1.f}, x, y, positions, wide, (int)L, (int)H, B * L,
                          dims[5], dims[6], dims[7], dims[8], dims[9], dims[10]};
    const auto launch = [&](auto kernel) {
        hipLaunchKernelGGL(kernel, dim3((unsigned)groups, (unsigned)((H + slice - 1) / slice)), dim3(ROW_WAVES * 64), 0, (hipStream_t)stream, a);
        return (int)hipGetLastError();
    };
    return type == RDA_FP16 ? launch(rotate_kernel<half_t>) : type == RDA_BF16 ? launch(rotate_kernel<bf16_t>) : launch(rotate_kernel<float>);
}

int rda_paged_append(const void* q, const void* k, const void* v, void* q_out, void* k_pages, void* v_pages, const int* table, const int* starts,
                     const int* lengths, const double* turns, float factor, int interleaved, int type, int cache_type, const long* dims, void* stream) {
    const long T = dims[0], H = dims[1], Hkv = dims[2], D = dims[3], R = dims[4], B = dims[5], N = dims[6], P = dims[8], S = dims[9];
    if (T <= 0 || T > MAX_ROWS || H < 0 || Hkv <= 0 || H + 2 * Hkv > 65535 || !rotary_ok(turns, D, R) || B <= 0 || B >= 1L << 30 || N <= 0 || P <= 0 || P >= 1L << 31 ||
        S <= 0 || N > ((1L << 31) - (1L << 16)) / S)
        return RDA_ERR_INVALID;
    if (type < RDA_FP16 || type > RDA_FP32 || cache_type < RDA_FP16 || cache_type > RDA_FP32) return RDA_ERR_INVALID;
    if (!vector_rows(k, dims + 12, 2, type) || !vector_rows(v, dims + 14, 2, type) || !vector_rows(k_pages, dims + 18, 3, cache_type) ||
        !vector_rows(v_pages, dims + 21, 3, cache_type))
        return RDA_ERR_INVALID;
    if (H && (!vector_rows(q, dims + 10, 2, type) || !vector_rows(q_out, dims + 16, 2, cache_type))) return RDA_ERR_INVALID;
    const AppendArgs a = {{turns, (int)D, (int)R, interleaved, factor, 1.f}, q, k, v, q_out, k_pages, v_pages, table, starts, lengths,
                          (int)T, (int)H, (int)Hkv, (int)B, (int)N, (int)P, make_div((int)S), dims[7], dims[10], dims[11], dims[12], dims[13], dims[14],
                          dims[15], dims[16], dims[17], dims[18], dims[19], dims[20], dims[21], dims[22], dims[23]};
    const long slice = 64 / (D / 16) * PASSES;
    const auto launch = [&](auto kernel) {
        hipLaunchKernelGGL(kernel, dim3((unsigned)((T + ROW_WAVES - 1) / ROW_WAVES), (unsigned)((H + 2 * Hkv + slice - 1) / slice)), dim3(ROW_WAVES * 64), 0,
                           (hipStream_t)stream, a);
        return (int)hipGetLastError();
    };
    const auto from = [&](auto x) {
        using X = decltype(x);
        return cache_type == RDA_FP16 ? launch(append_kernel<X, half_t>) : cache_type == RDA_BF16 ? launch(append_kernel<X, bf16_t>) : launch(append_kernel<X, float>);
    };
    return type == RDA_FP16 ? from(half_t{}) : type == RDA_BF16 ? from(bf16_t{}) : from(float{});
}

}  // extern "C"
