// A paged key/value cache held in 8 bits: values quantized as they are written, read back, and attention over them.
//
// Codes are int8; a block of 16, 32 or 64 consecutive tokens of a KV head has one scale in fp32 for its keys and one for its values: a value is
// code x scale, the scale the block's largest magnitude / 127. Pages are whole blocks, and blocks are whole groups of 16 tokens, so that 16 aligned keys
// share a page, a table entry and a scale. A scale that is not finite stands for a block of NaN, which is what values that are not all finite become.
#include "paged_work.h"
#include "rotary.h"

#define MAX_KEYS8 ((1L << 31) - (1L << 16))

// ------------------------------------------------------------------------------------------------ appending

struct Append8Args {
    RotaryArgs r;
    const void *q, *k, *v;
    void* qo;
    signed char *kc, *vc;
    float *ks, *vs;
    const int *table, *starts, *lengths;
    const void *qw, *kw;  // weights of the heads' norms, or null
    int wtype;
    float eps;
    int T, H, Hkv, B, N, P, block, slice;  // tokens of a block (16, 32, 64); heads of a workgroup
    Div S;
    long pitch, sqt, sqh, skt, skh, svt, svh, sot, soh, kpp, kpr, kph, vpp, vpr, vph, ksp, ksb, ksh, vsp, vsb, vsh;
};

// The last of B sequences that begins at or below `target` (B: behind them), its first row and the next one's, and its length; a sequence begins at
// key(starts[b], b). 64 are looked at in a step, one per lane, and the last step's lanes hold what is asked for of theirs, so that it costs one access to
// memory where there are at most 64.
struct Sequence {
    int b, first, end, length;
};
template <class Key>
__device__ __forceinline__ Sequence find_sequence(const int* starts, const int* lengths, int B, int target, int lane, Key&& key) {
    int at = 0, n = B;  // the answer is at .. at + n
    while (n > 64) {
        const int step = (n + 63) >> 6, i = (lane + 1) * step;
        const bool below = i <= n && key(starts[at + i], at + i) <= target;
        const int c = __popcll(__ballot(below));
        at += c * step;
        n = min(step - 1, n - c * step);
    }
    const int from = starts[min(at + lane, B)], to = starts[min(at + lane + 1, B)], length = lengths[min(at + lane, B - 1)];
    const bool below = lane < n && key(to, at + lane + 1) <= target;
    const int c = __builtin_amdgcn_readfirstlane(__popcll(__ballot(below)));
    Sequence s = {__builtin_amdgcn_readfirstlane(at) + c, 0, 0, 0};
    if (c < 64) {
        s.first = __builtin_amdgcn_readlane(from, c);
        s.end = __builtin_amdgcn_readlane(to, c);
        s.length = __builtin_amdgcn_readlane(length, c);
    } else if (s.b < B) {
        s.first = starts[s.b];
        s.end = starts[s.b + 1];
        s.length = lengths[s.b];
    }
    return s;
}

// Eight values or weights as they lie in memory, so that loads are not waited for where they are issued.
template <class X>
struct Raw8 {
    u4v v[sizeof(X) / 2];
    __device__ __forceinline__ void load(const X* p) {
#pragma unroll
        for (int i = 0; i < (int)(sizeof(X) / 2); i++) v[i] = ((const u4v*)p)[i];
    }
    __device__ __forceinline__ f8 values() const { return load8((const X*)v); }
};
struct RawWeights {
    u4v v[2];  // of 16-bit types the first alone
    __device__ __forceinline__ void load(const void* w, int type, int at) {
        const char* p = (const char*)w + at * (type == RDA_FP32 ? 4 : 2);
        v[0] = *(const u4v*)p;
        v[1] = *(const u4v*)(p + (type == RDA_FP32 ? 16 : 0));
    }
    __device__ __forceinline__ f8 values(int type) const { return weights8(v, type, 0); }
};

// The largest over the wave's lanes.
__device__ __forceinline__ u32 wave_max(u32 x) {
    x = max(x, (u32)__builtin_amdgcn_update_dpp(0, (int)x, 0xB1, 0xF, 0xF, true));
    x = max(x, (u32)__builtin_amdgcn_update_dpp(0, (int)x, 0x4E, 0xF, 0xF, true));
    x = max(x, (u32)__builtin_amdgcn_update_dpp(0, (int)x, 0x141, 0xF, 0xF, true));
    x = max(x, (u32)__builtin_amdgcn_update_dpp(0, (int)x, 0x140, 0xF, 0xF, true));
    const auto a = __builtin_amdgcn_permlane16_swap(x, x, false, false);
    x = max((u32)a[0], (u32)a[1]);
    const auto b = __builtin_amdgcn_permlane32_swap(x, x, false, false);
    return max((u32)b[0], (u32)b[1]);
}
__device__ __forceinline__ int to_code(float x) { return (int)rintf(fminf(fmaxf(x, -127.f), 127.f)); }
// Eight quotients as codes.
__device__ __forceinline__ void store_codes(signed char* p, const f8& x) {
    *(u2v*)p = (u2v){pack4(to_code(x[0]), to_code(x[1]), to_code(x[2]), to_code(x[3])), pack4(to_code(x[4]), to_code(x[5]), to_code(x[6]), to_code(x[7]))};
}
// x / s by 1 / s and one correction, to within an ulp: ties of values that 16 bits hold fall as those of the division do.
__device__ __forceinline__ f8 over(const f8& x, float s, float by) {
    f8 y;
#pragma unroll
    for (int e = 0; e < 8; e++) y[e] = div_by_scale(x[e], s, by);
    return y;
}
__device__ __forceinline__ f8 load_codes(const signed char* p) {
    const u2v w = *(const u2v*)p;
    f8 x;
#pragma unroll
    for (int i = 0; i < 8; i++) x[i] = (float)(int)(signed char)(w[i >> 2] >> (8 * (i & 3)));
    return x;
}
#define FLT_TOP 3.402823466e38f
#define LEAST_SCALE 1e-30f
// The largest magnitude of 16 values, as bits: magnitudes order as their bits do, infinities and NaN above the finite ones.
__device__ __forceinline__ u32 largest(const f8& a, const f8& b) {
    u32 top = 0;
#pragma unroll
    for (int e = 0; e < 8; e++) top = max(top, max(__float_as_uint(a[e]) & 0x7fffffffu, __float_as_uint(b[e]) & 0x7fffffffu));
    return top;
}
// The scale of a block whose new values' largest magnitude is `top` and whose older ones' scale is `had` (0: it has none): NaN, and codes of 0, where not all are finite.
struct NewScale {
    float now, by;
    bool finite;
};
__device__ __forceinline__ NewScale new_scale(u32 top, float had) {
    const bool finite = top < 0x7f800000u && had <= FLT_TOP;
    const float now = finite ? fmaxf(fmaxf(__uint_as_float(top) / 127.f, LEAST_SCALE), had) : __builtin_nanf("");
    return {now, finite ? 1.f / now : 0.f, finite};
}
// The largest over the `per` lanes that hold a head.
__device__ __forceinline__ u32 head_max(u32 x, int per, int lane) {
    if ((per & (per - 1)) == 0) {
        if (per >= 2) x = max(x, (u32)__builtin_amdgcn_update_dpp(0, (int)x, 0xB1, 0xF, 0xF, true));
        if (per >= 4) x = max(x, (u32)__builtin_amdgcn_update_dpp(0, (int)x, 0x4E, 0xF, 0xF, true));
        if (per >= 8) x = max(x, (u32)__builtin_amdgcn_update_dpp(0, (int)x, 0x141, 0xF, 0xF, true));
        if (per >= 16) x = max(x, (u32)__builtin_amdgcn_update_dpp(0, (int)x, 0x140, 0xF, 0xF, true));
        return x;
    }
    const int base = lane - lane % per;
    u32 top = 0;
    for (int i = 0; i < per; i++) top = max(top, (u32)__shfl((int)x, base + i));
    return top;
}

// One step's keys and values as codes into their blocks, keys normed and turned on the way, and queries normed and turned. A workgroup takes a block
// and `slice` heads (queries, keys, values in this order): it makes the angles of the block's new tokens once, and takes 16 tokens of a head to a wave, block / 16
// waves to a head. A block whose first tokens are older keeps a scale at least as large as it had; where the scale grows the older codes are
// rounded anew to it by the same workgroup, which alone writes the block of that head.
//
// The loads of the next heads go out ahead of the arithmetic on these. 16384 tokens of 32 + 2 x 8 heads of 128 fp16 with norms, 369 MB: 90 us, 4.1 TB/s, vector work
// 44% of the cycles; 3 ragged chunks of fp32, 43 MB: 13.7 us.
template <class X, class Q, int PS>
__global__ __launch_bounds__(256) void append8_kernel(Append8Args p) {
    extern __shared__ __attribute__((aligned(16))) char smem[];
    __shared__ u32 most[2][4];
    f2* cs = (f2*)smem;  // [row of the block][pair]
    const int t = threadIdx.x, lane = t & 63, wave = __builtin_amdgcn_readfirstlane(t >> 6);
    const int pairs = p.r.R / 2, rows_at_once = pairs ? 256 / pairs : 0, my_pair = pairs ? t % pairs : 0;  // of the angles: a thread's pair stays
    const double turns = pairs ? p.r.turns[my_pair] : 0.;
    const int slot = blockIdx.x, shift = p.block == 16 ? 4 : p.block == 32 ? 5 : 6;
    // Sequence b's slots are those from here on: with its n new tokens it touches at most (n - 2) / block + 2 blocks, and has n / block rounded down
    // + 2 slots at least, whatever its position, so that no sums over the sequences are needed.
    auto first_slot = [&](int start, int b) __attribute__((always_inline)) { return (min(max(start, 0), p.T) >> shift) + 2 * b; };
    const Sequence q = find_sequence(p.starts, p.lengths, p.B, slot, lane, first_slot);
    if (q.b >= p.B) return;
    const int first = min(max(q.first, 0), p.T), tokens = min(max(q.end, first), p.T) - first;
    if (tokens == 0) return;
    const int p0 = max(q.length, -(1 << 30)) - tokens;  // position of the first new token; negative: no place for it
    const int b0 = ((p0 >> shift) + (slot - first_slot(q.first, q.b))) << shift;  // the block's first position
    const int o0 = max(p0 - b0, 0), o1 = min(p0 + tokens - b0, p.block);  // its new rows
    if (o0 >= o1) return;
    const int head0 = blockIdx.y * p.slice, head1 = min(head0 + p.slice, p.H + 2 * p.Hkv);
    const int entry = b0 >= 0 ? div_by(b0, p.S) : p.N;
    int page = -1;
    if (entry < p.N) page = p.table[q.b * p.pitch + entry];

    const Place pl = place(p.r, lane);
    const int per = p.r.D / 16, waves = p.block >> 4, sub = wave & (waves - 1), together = 4 / waves;  // waves of a head; the wave's 16 rows; heads at once
    int row[PS];
    bool mine[PS];
#pragma unroll
    for (int i = 0; i < PS; i++) {
        const int x = i * pl.heads + pl.head;
        row[i] = 16 * sub + x;
        mine[i] = pl.head < pl.heads && x < 16 && row[i] >= o0 && row[i] < o1;
    }
    // The values and weights of the wave's head of the heads h0 on, and the scale that its block has.
    Raw8<X> raw_lo[PS], raw_hi[PS];
    RawWeights raw_wl, raw_wh;
    float *raw_scale = nullptr, raw_had = 0.f;
    auto load = [&](int h0) __attribute__((always_inline)) {
        const int h = min(h0 + wave / waves, head1 - 1), hk = h - p.H, hv = hk - p.Hkv;
        const X* src = hk < 0 ? (const X*)p.q + h * p.sqh : hv < 0 ? (const X*)p.k + hk * p.skh : (const X*)p.v + hv * p.svh;
        const long st = hk < 0 ? p.sqt : hv < 0 ? p.skt : p.svt;
#pragma unroll
        for (int i = 0; i < PS; i++) {
            const X* at = src + (first + b0 - p0 + (mine[i] ? row[i] : o0)) * st;
            raw_lo[i].load(at + pl.at);
            raw_hi[i].load(at + pl.to);
        }
        if (p.kw && hv < 0) {
            raw_wl.load(hk < 0 ? p.qw : p.kw, p.wtype, pl.at);
            raw_wh.load(hk < 0 ? p.qw : p.kw, p.wtype, pl.to);
        }
        if (page >= 0 && page < p.P && hk >= 0) {
            const int part = (b0 - entry * (int)p.S.d) >> shift;  // the block's number in its page
            raw_scale = hv < 0 ? p.ks + page * p.ksp + part * p.ksb + hk * p.ksh : p.vs + page * p.vsp + part * p.vsb + hv * p.vsh;
            if (o0 > 0) raw_had = *raw_scale;
        }
    };
    load(head0);
    const bool there = page >= 0 && page < p.P;
    const int row0 = there ? b0 - entry * (int)p.S.d : 0;  // the block's first row of the page

    if (pairs && head0 < p.H + p.Hkv) {
        if (t < rows_at_once * pairs)
            for (int row = o0 + t / pairs; row < o1; row += rows_at_once) {
                const f2 v = cos_sin((double)(b0 + row), turns);
                cs[row * pairs + my_pair] = (f2){v[0] * p.r.factor, v[1] * p.r.factor};
            }
        __syncthreads();
    }
    int turn_of = 0;
    for (int h0 = head0; h0 < head1; h0 += together, turn_of ^= 1) {
        const int h = h0 + wave / waves, hk = h - p.H, hv = hk - p.Hkv;
        const bool active = h < head1, writes = active && hk >= 0 && there;
        float* const scale = raw_scale;
        const float had = raw_had;
        f8 lo[PS], hi[PS];
        if (active) {
#pragma unroll
            for (int i = 0; i < PS; i++) {
                lo[i] = raw_lo[i].values();
                hi[i] = raw_hi[i].values();
            }
            if (p.kw && hv < 0) {
                const f8 wl = raw_wl.values(p.wtype), wh = raw_wh.values(p.wtype);
#pragma unroll
                for (int i = 0; i < PS; i++) {
                    const float inv = inverse_rms(lo[i], hi[i], p.r.D, p.eps, per, lane);
                    lo[i] = lo[i] * inv * wl;
                    hi[i] = hi[i] * inv * wh;
                }
            }
            if (hv < 0 && pl.pair >= 0) {
#pragma unroll
                for (int i = 0; i < PS; i++) {
                    f8 c, s;
                    angles_of(pl, cs + (mine[i] ? row[i] : o0) * pairs, c, s);
                    turn(lo[i], hi[i], c, s, p.r.interleaved);
                }
            }
            if (h0 + together < head1) load(h0 + together);
            if (hk < 0) {
#pragma unroll
                for (int i = 0; i < PS; i++)
                    if (mine[i]) {
                        Q* dst = (Q*)p.qo + (long)(first + b0 - p0 + row[i]) * p.sot + h * p.soh;
                        store8(dst + pl.at, lo[i]);
                        store8(dst + pl.to, hi[i]);
                    }
            }
        }
        if (h0 + together <= p.H) continue;  // queries all (the same for the workgroup)
        u32 top = 0;  // magnitudes order as their bits do, infinities and NaN above the finite ones
        if (active && hk >= 0) {
#pragma unroll
            for (int i = 0; i < PS; i++)
                if (mine[i]) top = max(top, largest(lo[i], hi[i]));
            top = wave_max(top);
        }
        if (waves > 1) {  // also: every wave has read the scale before one writes it
            if (lane == 0) most[turn_of][wave] = top;
            __syncthreads();
            for (int i = wave & ~(waves - 1), n = i + waves; i < n; i++) top = max(top, most[turn_of][i]);
        }
        if (!writes) continue;
        signed char* codes = hv < 0 ? p.kc + page * p.kpp + row0 * p.kpr + hk * p.kph : p.vc + page * p.vpp + row0 * p.vpr + hv * p.vph;
        const long cr = hv < 0 ? p.kpr : p.vpr;
        const NewScale s = new_scale(top, had);
#pragma unroll
        for (int i = 0; i < PS; i++) {
            if (mine[i]) {
                store_codes(codes + row[i] * cr + pl.at, s.finite ? over(lo[i], s.now, s.by) : (f8){});
                store_codes(codes + row[i] * cr + pl.to, s.finite ? over(hi[i], s.now, s.by) : (f8){});
            }
        }
        if (o0 > 0 && s.finite && s.now != had) {
            const float shrink = had * s.by;
#pragma unroll
            for (int i = 0; i < PS; i++) {
                const int x = i * pl.heads + pl.head;
                if (pl.head < pl.heads && x < 16 && row[i] < o0) {
                    signed char* at = codes + row[i] * cr;
                    const f8 a = load_codes(at + pl.at), z = load_codes(at + pl.to);
                    store_codes(at + pl.at, a * shrink);
                    store_codes(at + pl.to, z * shrink);
                }
            }
        }
        if (sub == 0 && lane == 0) *scale = s.now;
    }
}

// The same for steps of few tokens a sequence, whose blocks have one new row, seldom more: a wave takes a token and as many heads of one tensor as its lanes
// hold, 16 values each. A block's new keys and values are written by the wave of its first new token, which goes over the others once for the
// largest value and once to write them. (The kernel above runs a wave for each head of a block here: 14.4 us for 64 single
// tokens of 32 + 2 x 8 heads, this one 4.5; 11.1 where the keys of every block, 31 rows, are rounded anew.)
template <class X, class Q>
__global__ __launch_bounds__(256) void append8_few_kernel(Append8Args p) {
    __shared__ __attribute__((aligned(16))) f2 cs_all[4][MAX_PAIRS];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    f2* cs = cs_all[wave];
    const int pairs = p.r.R / 2, shift = p.block == 16 ? 4 : p.block == 32 ? 5 : 6;
    double f0 = 0, f1 = 0;
    if (pairs) {
        f0 = p.r.turns[min(lane, pairs - 1)];
        f1 = p.r.turns[min(lane + 64, pairs - 1)];
    }
    const Place pl = place(p.r, lane);
    const int per = p.r.D / 16;
    // Workgroup y: slices of the query heads, of the key heads, of the value heads, four of them to its waves.
    const int qs = (p.H + pl.heads - 1) / pl.heads, ks = (p.Hkv + pl.heads - 1) / pl.heads, slice = blockIdx.y * 4 + wave;
    if (slice >= qs + 2 * ks) return;
    const int kind = slice < qs ? 0 : slice < qs + ks ? 1 : 2, heads = kind ? p.Hkv : p.H;
    const int h = (slice - (kind == 0 ? 0 : kind == 1 ? qs : qs + ks)) * pl.heads + pl.head;
    const bool mine = pl.head < pl.heads && h < heads;
    const int hc = mine ? h : 0;
    const X* src = kind == 0 ? (const X*)p.q + hc * p.sqh : kind == 1 ? (const X*)p.k + hc * p.skh : (const X*)p.v + hc * p.svh;
    const long st = kind == 0 ? p.sqt : kind == 1 ? p.skt : p.svt;
    const void* w = kind == 0 ? p.qw : kind == 1 ? p.kw : nullptr;
    const int token = blockIdx.x;
    Raw8<X> raw_lo, raw_hi;
    RawWeights raw_wl, raw_wh;
    raw_lo.load(src + token * st + pl.at);
    raw_hi.load(src + token * st + pl.to);
    if (w) {
        raw_wl.load(w, p.wtype, pl.at);
        raw_wh.load(w, p.wtype, pl.to);
    }
    const Sequence q = find_sequence(p.starts, p.lengths, p.B, token, lane, [](int start, int) { return start; });
    if (q.b >= p.B || token < q.first) return;
    const int first = max(q.first, 0), end = min(max(q.end, first), p.T);
    const int n = max(q.length, -(1 << 30)) - (end - token);  // the token's position
    const int b0 = (n >> shift) << shift, entry = b0 >= 0 ? div_by(b0, p.S) : p.N;
    int rows = 1;  // of the block's new ones, from this one on
    if (kind) {
        if (token > first && n > b0) return;  // not the block's first new token
        rows = min(end - token, p.block - (n - b0));
    }
    int page = -1;
    if (kind && entry < p.N) page = p.table[q.b * p.pitch + entry];
    if (kind && (page < 0 || page >= p.P)) return;
    const int o0 = n - b0;
    signed char* codes = nullptr;
    float *scale = nullptr, had = 0.f;
    long cr = 0;
    if (kind) {
        const int row0 = b0 - entry * (int)p.S.d, part = row0 >> shift;
        codes = kind == 1 ? p.kc + page * p.kpp + row0 * p.kpr + hc * p.kph : p.vc + page * p.vpp + row0 * p.vpr + hc * p.vph;
        scale = kind == 1 ? p.ks + page * p.ksp + part * p.ksb + hc * p.ksh : p.vs + page * p.vsp + part * p.vsb + hc * p.vsh;
        cr = kind == 1 ? p.kpr : p.vpr;
        if (o0 > 0) had = *scale;
    }
    u32 top = 0;
    NewScale s = {};
    for (int it = 0, all = rows == 1 ? 1 : 2 * rows; it < all; it++) {
        const int i = it < rows ? it : it - rows;
        if (it > 0) {
            raw_lo.load(src + (token + i) * st + pl.at);
            raw_hi.load(src + (token + i) * st + pl.to);
        }
        f8 lo = raw_lo.values(), hi = raw_hi.values();
        if (w) {
            const float inv = inverse_rms(lo, hi, p.r.D, p.eps, per, lane);
            lo = lo * inv * raw_wl.values(p.wtype);
            hi = hi * inv * raw_wh.values(p.wtype);
        }
        if (pairs && kind < 2) {
            __builtin_amdgcn_wave_barrier();  // the last token's angles have been read
            make_angles(p.r, f0, f1, (double)(n + i), cs, lane);
            f8 c, sn;
            angles_of(pl, cs, c, sn);
            if (pl.pair >= 0) turn(lo, hi, c, sn, p.r.interleaved);
        }
        if (kind == 0) {
            if (mine) {
                Q* dst = (Q*)p.qo + token * p.sot + h * p.soh;
                store8(dst + pl.at, lo);
                store8(dst + pl.to, hi);
            }
            return;
        }
        if (it < rows) top = max(top, largest(lo, hi));
        if (it == rows - 1) {
            s = new_scale(head_max(top, per, lane), had);
            if (mine && o0 > 0 && s.finite && s.now != had) {
                const float shrink = had * s.by;
                for (int r = 0; r < o0; r += 8) {  // eight rows' loads ahead of their stores
                    f8 a[8], z[8];
#pragma unroll
                    for (int x = 0; x < 8; x++) {
                        const signed char* at = codes + min(r + x, o0 - 1) * cr;
                        a[x] = load_codes(at + pl.at);
                        z[x] = load_codes(at + pl.to);
                    }
#pragma unroll
                    for (int x = 0; x < 8; x++)
                        if (r + x < o0) {
                            store_codes(codes + (r + x) * cr + pl.at, a[x] * shrink);
                            store_codes(codes + (r + x) * cr + pl.to, z[x] * shrink);
                        }
                }
            }
            if (mine && lane % per == 0) *scale = s.now;
        }
        if (mine && it >= all - rows) {
            store_codes(codes + (o0 + i) * cr + pl.at, s.finite ? over(lo, s.now, s.by) : (f8){});
            store_codes(codes + (o0 + i) * cr + pl.to, s.finite ? over(hi, s.now, s.by) : (f8){});
        }
    }
}

// ------------------------------------------------------------------------------------------------ reading back

struct Read8Args {
    const signed char *kc, *vc;
    const float *ks, *vs;
    const int *table, *starts, *lengths;
    void *ko, *vo;
    int T, Hkv, D, B, N, P, shift;
    Div S;
    long pitch, kpp, kpr, kph, vpp, vpr, vph, ksp, ksb, ksh, vsp, vsb, vsh;
};

// Keys and values of a batch's rows as the values that their codes stand for: a wave takes a row, its lanes 16 values each. Rows of no
// sequence, and of positions that the cache does not have, are 0. Bound by memory: 24 sequences, 160 MB, 32 us, 4.9 TB/s; 257 rows 4 us, three accesses to memory one
// after the other.
template <class X>
__global__ __launch_bounds__(256) void read8_kernel(Read8Args p) {
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), token = blockIdx.x * 4 + wave;
    if (token >= p.T) return;
    const Sequence q = find_sequence(p.starts, p.lengths, p.B, token, lane, [](int start, int) { return start; });
    int page = -1, row = 0;
    if (q.b < p.B && token >= q.first) {
        const long n = (long)q.length - q.end + token;
        const int entry = n >= 0 && n < 1L << 31 ? div_by((int)n, p.S) : p.N;
        if (entry < p.N) page = p.table[q.b * p.pitch + entry], row = (int)n - entry * (int)p.S.d;
    }
    const bool there = page >= 0 && page < p.P;
    const int per = p.D / 16, chunks = p.Hkv * per;
    for (int i = lane; i < 2 * chunks; i += 64) {
        const bool value = i >= chunks;
        const int c = value ? i - chunks : i, h = c / per, at = c % per * 16;
        f8 lo = {}, hi = {};
        if (there) {
            const signed char* src = (value ? p.vc + page * p.vpp + row * p.vpr + h * p.vph : p.kc + page * p.kpp + row * p.kpr + h * p.kph) + at;
            const float scale = value ? p.vs[page * p.vsp + (row >> p.shift) * p.vsb + h * p.vsh] : p.ks[page * p.ksp + (row >> p.shift) * p.ksb + h * p.ksh];
            const float by = scale <= FLT_TOP ? scale : __builtin_nanf("");
            lo = load_codes(src) * by;
            hi = load_codes(src + 8) * by;
        }
        X* dst = (X*)(value ? p.vo : p.ko) + ((long)token * p.Hkv + h) * p.D + at;
        store8(dst, lo);
        store8(dst + 8, hi);
    }
}

// ------------------------------------------------------------------------------------------------ attention

struct Attn8Args : PagedArgs {
    const float *ks, *vs;
    u32 ksp, ksb, vsp, vsb;  // strides of pages and of blocks of the scales
    long ksh, vsh;
    int shift;  // log2 of a block's tokens
    int spread;  // whether each XCD takes parts of all KV heads
};
#define LIFT8 7.f  // P stands 2^7 above 2^(x - m), so that it may be 2^15 where m lags by 8

// Codes as fp16: byte b, its sign bit flipped, in the low byte of 0x6400 is 1024 + 128 + code; less 1152 it is the code, exactly.
__device__ __forceinline__ u32 less_bias(u32 w) {
    return __builtin_bit_cast(u32, __builtin_bit_cast(h2, w) + (h2){(half_t)-1152.f, (half_t)-1152.f});
}
__device__ __forceinline__ u2v widen4(u32 w) {
    w ^= 0x80808080u;
    return (u2v){less_bias(__builtin_amdgcn_perm(0x64646464u, w, 0x04010400u)), less_bias(__builtin_amdgcn_perm(0x64646464u, w, 0x04030402u))};
}
// Byte j (a constant) of a and of b, their sign bits flipped before, as two fp16 codes x 2^-9: a byte in the low half of a word is the fp16 byte x 2^-24; that
// times 2^15, less 128 x 2^-9 in the same operation, is exact.
__device__ __forceinline__ u32 widen_pair(u32 a, u32 b, int j) {
    const h2 x = __builtin_bit_cast(h2, __builtin_amdgcn_perm(b, a, 0x0c000c00u | (u32)j | (u32)(4 + j) << 16));
    return __builtin_bit_cast(u32, __builtin_elementwise_fma(x, (h2){(half_t)32768.f, (half_t)32768.f}, (h2){(half_t)-0.25f, (half_t)-0.25f}));
}
__device__ __forceinline__ f4 product16(const u4v& a, const u4v& b, const f4& c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(h8, a), __builtin_bit_cast(h8, b), c, 0, 0, 0);
}

// Tiles of 16 MB rows, as rows_kernel of 16-bit caches (paged_attention.hip) has them, in units of 256 keys: a wave's tile is 64 keys, lane
// group g = l / 16 holding the scores of keys 16 g .. 16 g + 15 (score block c's row 4 g + i stands for key 16 g + 4 c + i), which share a page and a
// scale of K and of V. All products are of fp16: codes are exact there, and a row of q is brought to a largest magnitude of 2^14 to 2^15 by a power
// of two that its scores' factor takes back (a bf16 value less than 2^-28 of its row's largest may lose bits). P is what the scale of V leaves of
// it relative to the largest scale that the row has met, vm: O is in units of vm, and rescaled when that grows, as when the maximum moves. l sums P
// before both: P and its sum are then off by roundings of P to fp16 that do not cancel, up to 1.3 times the rms error of a plain form that keeps P in 32 bits (fp16
// outputs; with bf16 ones the output's rounding hides it).
//
// Bound by the keys and values read: 64 single tokens over 8192 keys (8 KV heads of 128), 1.08 GB, 206 to 209 us, 5.2 TB/s, in pages of whole heads 188, 5.7, where a large sum
// reads at 6.0; vector work, half of it widening codes, takes 33% of the cycles. Loads are issued in the order in which they are waited for: each wait is then for
// its own loads alone, with the next tile's 16 KiB (of K, then of V) behind them.
//
// Tiles of 32 rows take 32 keys a wave (64 spill registers: 32 sequences of 5 tokens over 4096 keys 67.5 us, 61.6 so); tiles of 16 rows 64 (with 32: 64 x 8192 213 us, 209
// so, and at three workgroups a CU 219, where 61 ragged sequences gain 5%).
__host__ __device__ constexpr int rows8_steps(int mb) { return mb == 1 ? 2 : 1; }  // 32 keys each
template <class T, int D, int MB, bool MOD>
__global__ __launch_bounds__(256, 2) void rows8_kernel(Attn8Args p) {
    constexpr int NS = rows8_steps(MB), KT = 32 * NS, KG = 8 * NS, UK = 4 * KT, MT = 16 * MB, AHEAD = ahead(MT, MOD);
    constexpr int KC = D / 64;  // 16-byte vectors of a lane's part of a K row
    constexpr int VC = D / 16;  // consecutive dims of a lane's part of a V row
    constexpr int OP = D + 4;   // pitch of a row of O in LDS
    typedef typename std::conditional<VC == 8, u2v, u32>::type vvec;
    extern __shared__ __attribute__((aligned(16))) char smem[];
    __shared__ u32 shared[256 + 8];
    __shared__ float ml[2][4][16];
    const int t = threadIdx.x, lane = t & 63, g = lane >> 4, r = lane & 15;
    const int wave = __builtin_amdgcn_readfirstlane(t >> 6);
    const int block = p.spread ? (int)blockIdx.x : work_block(p.grid);
    Run run = find_run<MT, UK, AHEAD, 256, true>(p, (int*)smem, shared, block);
    Cut cut = {};

    while (run.count > 0) {
        const WorkTile w = uniform(make_tile<MT, UK, AHEAD, true>(p, run.b, run.j));
        if (run.unit + run.count <= AHEAD) break;  // the next run's
        const bool begins = run.unit == 0, last_part = run.unit + run.count >= w.units, whole = begins && last_part;
        const int u0 = begins ? 0 : run.unit - AHEAD, u1 = min(w.units, run.unit + run.count) - AHEAD, n = u1 - u0;
        const int* table = p.table + run.b * p.pitch;
        const signed char* kbase = (const signed char*)p.k + run.kvh * p.kph;
        const signed char* vbase = (const signed char*)p.v + run.kvh * p.vph;
        const float *ksbase = p.ks + run.kvh * p.ksh, *vsbase = p.vs + run.kvh * p.vsh;

        const int n0 = uniform(w.p0 + div_by(w.r0, p.G)), n1 = uniform(w.p0 + div_by(w.r1, p.G));

        f4 o[MB][VC];
        float m_[MB], l_[MB], vm[MB];
#pragma unroll
        for (int m = 0; m < MB; m++) {
#pragma unroll
            for (int j = 0; j < VC; j++) o[m][j] = (f4){};
            m_[m] = -__builtin_inff();
            l_[m] = 0.f;
            vm[m] = 1e-36f;  // 128 / vm stays finite
        }

        if (w.hi > w.lo) {
            const int last = (w.hi - 1) / KG * KG;
            auto key_of = [&](int i) __attribute__((always_inline)) { return w.lo + (u0 + i) * UK + (u0 + i >= w.head ? w.skip : 0) + wave * KT; };
            // Table entries of the lane's K rows and of its keys of V: of tile i + 1 until its loads of K, then of tile i + 2. What is waited for first is
            // loaded first: scales and table entries ahead of V, whose loads end a step.
            int kid, vid;
            auto fetch_ids = [&](int i) __attribute__((always_inline)) {
                const int key0 = key_of(i);
                kid = table[div_by(min(key0 + KG * (r >> 2), last), p.S)];
                vid = table[div_by(min(key0 + KG * g, last), p.S)];
            };
            u4v kf[KG / 4][KC];
            vvec vf[KG];
            float ks, vs, ks2, vs2;  // the scales of the lane's keys, of tile i and of tile i + 1
            u32 vrow, vpage;         // where V of tile i + 1 lies
            bool bad = false, bad2;  // the lane's keys are on a page that the cache does not have
            auto load_k = [&](int i) __attribute__((always_inline)) {
                const int vkey = min(key_of(i) + KG * g, last), key = min(key_of(i) + KG * (r >> 2), last), row = key - div_by(key, p.S) * (int)p.S.d + (r & 3);
                vrow = (u32)(vkey - div_by(vkey, p.S) * (int)p.S.d);
                bad2 = (u32)vid >= (u32)p.P;
                vpage = bad2 ? 0 : (u32)vid;
                ks2 = ksbase[row_at(vpage, p.ksp, vrow >> p.shift, p.ksb)];
                vs2 = vsbase[row_at(vpage, p.vsp, vrow >> p.shift, p.vsb)];
                const signed char* src = kbase + row_at((u32)kid < (u32)p.P ? (u32)kid : 0, p.kpp, (u32)row, p.kpr) + 16 * g;
#pragma unroll
                for (int c = 0; c < KG / 4; c++)
#pragma unroll
                    for (int x = 0; x < KC; x++) kf[c][x] = *(const u4v*)(src + (unsigned long long)(4 * c) * p.kpr + 64 * x);
            };
            auto load_v = [&]() __attribute__((always_inline)) {
                const signed char* src = vbase + row_at(vpage, p.vpp, vrow, p.vpr) + r * VC;
#pragma unroll
                for (int e = 0; e < KG; e++) vf[e] = *(const vvec*)(src + (unsigned long long)e * p.vpr);
                ks = ks2;
                vs = vs2;
                bad = bad2;
            };
            // A run's start is a chain of accesses to memory, each waited for behind those that it does not need: table entries, Q, then keys and values.
            fetch_ids(0);
            // Q as the B operand: lane (g, r) has values 64 x + 16 g .. + 15 of row r, as it has of the K rows.
            u4v qf[MB][KC][2];
            int pos[MB], pre[MB];
            float slope[MB], by[MB];  // by: what a product is times, but the key's scale
#pragma unroll
            for (int m = 0; m < MB; m++) {
                const int row = w.r0 + 16 * m + r, rc = min(row, w.r1), token = div_by(rc, p.G), head = run.kvh * (int)p.G.d + rc - token * (int)p.G.d;
                const T* src = (const T*)p.q + (long)(w.first + token) * p.sqt + head * p.sqh;
#pragma unroll
                for (int c = 0; c < KC; c++)
#pragma unroll
                    for (int h = 0; h < 2; h++) qf[m][c][h] = *(const u4v*)(src + 64 * c + 16 * g + 8 * h);
                pos[m] = row <= w.r1 ? w.p0 + token : -1;
                pre[m] = row <= w.r1 ? w.prefix : 0;
                slope[m] = MOD && p.slopes ? p.slopes[head] * LOG2E : 0.f;
            }
            __builtin_amdgcn_sched_barrier(0);
            load_k(0);
            fetch_ids(min(1, n - 1));
            __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int m = 0; m < MB; m++) {
                f8 x[KC][2];
                float top = 0.f;
#pragma unroll
                for (int c = 0; c < KC; c++)
#pragma unroll
                    for (int h = 0; h < 2; h++) {
                        x[c][h] = load8((const T*)&qf[m][c][h]);
#pragma unroll
                        for (int e = 0; e < 8; e++) top = fmaxf(top, fabsf(x[c][h][e]));
                    }
                top = rows_max(top);
                const int up = top > 0.f && top <= FLT_TOP ? 15 - __builtin_amdgcn_frexp_expf(top) : 0;
                by[m] = ldexpf(p.scale, -up);
#pragma unroll
                for (int c = 0; c < KC; c++)
#pragma unroll
                    for (int h = 0; h < 2; h++) {
#pragma unroll
                        for (int e = 0; e < 8; e++) x[c][h][e] = ldexpf(x[c][h][e], up);
                        qf[m][c][h] = __builtin_bit_cast(u4v, __builtin_convertvector(x[c][h], h8));
                    }
            }
            load_v();
            for (int i = 0;; i++) {
                const int key0 = key_of(i);
                if (!(ks <= FLT_TOP)) ks = __builtin_nanf("");
                float s[MB][KG];
#pragma unroll
                for (int c = 0; c < KG / 4; c++) {
                    u4v a[KC][2];
#pragma unroll
                    for (int x = 0; x < KC; x++)
#pragma unroll
                        for (int h = 0; h < 2; h++) {
                            const u2v lo = widen4(kf[c][x][2 * h]), hi = widen4(kf[c][x][2 * h + 1]);
                            a[x][h] = (u4v){lo[0], lo[1], hi[0], hi[1]};
                        }
#pragma unroll
                    for (int m = 0; m < MB; m++) {
                        f4 acc = {};
#pragma unroll
                        for (int x = 0; x < KC; x++)
#pragma unroll
                            for (int h = 0; h < 2; h++) acc = product16(a[x][h], qf[m][x][h], acc);
                        const float f = by[m] * ks;
#pragma unroll
                        for (int e = 0; e < 4; e++) s[m][4 * c + e] = acc[e] * f;
                    }
                }
                const bool hole = bad;
                // (The last tile's K again behind it, from L2: under a branch the waits for V would be for these loads too.)
                load_k(min(i + 1, n - 1));
                fetch_ids(min(i + 2, n - 1));
                // Whether every row sees every key of the tile.
                const bool all = key0 + KT <= w.hi && !__any(hole) && (key0 + KT <= n0 + 1 || key0 + KT <= w.prefix) &&
                                 (p.window <= 0 || n1 - key0 < p.window || key0 + KT <= w.prefix);
                if constexpr (MOD) {
                    const auto cap_all = [&](auto fine) __attribute__((always_inline)) {
#pragma unroll
                        for (int m = 0; m < MB; m++)
#pragma unroll
                            for (int e = 0; e < KG; e++) s[m][e] = capped<decltype(fine)::value>(s[m][e], p.cap);
                    };
                    if (p.cap >= HIGH_CAP) cap_all(std::true_type{});
                    else if (p.cap > 0.f) cap_all(std::false_type{});
#pragma unroll
                    for (int m = 0; m < MB; m++)
#pragma unroll
                        for (int e = 0; e < KG; e++) s[m][e] = __builtin_fmaf(-slope[m], fabsf((float)(pos[m] - (key0 + KG * g + e))), s[m][e]);
                }
                u32 see[MB];
#pragma unroll
                for (int m = 0; m < MB; m++) see[m] = (1u << KG) - 1;
                if (!all) {
#pragma unroll
                    for (int m = 0; m < MB; m++) {
                        see[m] = 0;
#pragma unroll
                        for (int e = 0; e < KG; e++) {
                            const int key = key0 + KG * g + e;
                            const bool ok = key < w.hi && !hole && ((key <= pos[m] && (p.window <= 0 || pos[m] - key < p.window)) || key < pre[m]);
                            if (!ok) s[m][e] = -__builtin_inff();
                            see[m] |= ok ? 1u << e : 0;
                        }
                    }
                }
                // Softmax.
                u4v pf[MB][NS];
                const bool finite = vs <= FLT_TOP;
#pragma unroll
                for (int m = 0; m < MB; m++) {
                    float mx = s[m][0];
#pragma unroll
                    for (int e = 1; e < KG; e++) mx = fmaxf(mx, s[m][e]);
                    mx = rows_max(mx);
                    const float mine = see[m] && finite ? vs : 0.f, vx = rows_max(mine);
                    const bool move = mx > m_[m] + 8.f || (m_[m] == -__builtin_inff() && mx > m_[m]), grow = vx > vm[m];
                    if (__any(move || grow)) {
                        const float a = move ? __builtin_amdgcn_exp2f(m_[m] - mx) : 1.f, b = grow ? vm[m] / vx : 1.f;
                        m_[m] = move ? mx : m_[m];
                        vm[m] = grow ? vx : vm[m];
                        l_[m] *= a;
#pragma unroll
                        for (int j = 0; j < VC; j++) o[m][j] *= a * b;
                    }
                    if (see[m] && !finite) l_[m] = __builtin_nanf("");
                    const float base = m_[m] == -__builtin_inff() ? 0.f : m_[m], f = mine * (128.f / vm[m]);
                    float pw[KG];
#pragma unroll
                    for (int e = 0; e < KG; e++) pw[e] = __builtin_amdgcn_exp2f(s[m][e] - base);
#pragma unroll
                    for (int e = 0; e < KG; e++) l_[m] += pw[e];
#pragma unroll
                    for (int h = 0; h < NS; h++) {
                        h8 x;
#pragma unroll
                        for (int e = 0; e < 8; e++) x[e] = (half_t)(pw[8 * h + e] * f);
                        pf[m][h] = __builtin_bit_cast(u4v, x);
                    }
                }
                // O^T += V^T P^T.
#pragma unroll
                for (int e = 0; e < KG; e++) vf[e] ^= 0x80808080u;
#pragma unroll
                for (int j = 0; j < VC; j++)
#pragma unroll
                    for (int h = 0; h < NS; h++) {
                        u4v a;
#pragma unroll
                        for (int e = 0; e < 4; e++) {
                            u32 v0, v1;
                            if constexpr (VC == 8) v0 = vf[8 * h + 2 * e][j >> 2], v1 = vf[8 * h + 2 * e + 1][j >> 2];
                            else v0 = vf[8 * h + 2 * e], v1 = vf[8 * h + 2 * e + 1];
                            a[e] = widen_pair(v0, v1, j & 3);
                        }
#pragma unroll
                        for (int m = 0; m < MB; m++) o[m][j] = product16(a, pf[m][h], o[m][j]);
                    }
                if (i + 1 >= n) break;
                load_v();
            }
        }

        // The four waves' results meet in LDS, 16 rows at a time: thread (row t / 16, dims from t % 16 on) adds them.
#pragma unroll
        for (int m = 0; m < MB; m++) {
            const float l = rows_sum(l_[m]), unit = vm[m] * 4.f;  // P's 2^7, codes' 2^-9
            __syncthreads();
            if (g == 0) {
                ml[0][wave][r] = m_[m];
                ml[1][wave][r] = l;
            }
            float* dst = (float*)smem + (wave * 16 + r) * OP;
#pragma unroll
            for (int i = 0; i < 4; i++)  // dims VC (4 g + i) + j
#pragma unroll
                for (int j = 0; j < VC; j += 4)
                    *(f4*)(dst + VC * (4 * g + i) + j) = (f4){o[m][j][i], o[m][j + 1][i], o[m][j + 2][i], o[m][j + 3][i]} * unit;
            __syncthreads();
            const int row = t >> 4, c = (t & 15) * (D / 16);
            float top = ml[0][0][row];
#pragma unroll
            for (int x = 1; x < 4; x++) top = fmaxf(top, ml[0][x][row]);
            float sum = 0.f, y[D / 16];
#pragma unroll
            for (int e = 0; e < D / 16; e++) y[e] = 0.f;
#pragma unroll
            for (int x = 0; x < 4; x++) {
                const float a = ml[0][x][row] == -__builtin_inff() ? 0.f : __builtin_amdgcn_exp2f(ml[0][x][row] - top);
                sum = __builtin_fmaf(ml[1][x][row], a, sum);
                const float* src = (const float*)smem + (x * 16 + row) * OP + c;
#pragma unroll
                for (int e = 0; e < D / 16; e += 4) {
                    const f4 z = *(const f4*)(src + e);
#pragma unroll
                    for (int k = 0; k < 4; k++) y[e + k] = __builtin_fmaf(z[k], a, y[e + k]);
                }
            }
            const int tr = 16 * m + row;
            if (whole) {
                if (w.r0 + tr <= w.r1) {
                    const int token = div_by(w.r0 + tr, p.G), head = run.kvh * (int)p.G.d + w.r0 + tr - token * (int)p.G.d;
                    T* out = (T*)p.o + (long)(w.first + token) * p.sot + head * p.soh + c;
                    store_row<T, D>(out, y, sum);
                }
            } else {
                float* part = partial<MT, D>(p, block, begins);
#pragma unroll
                for (int e = 0; e < D / 16; e += 4) *(f4*)(part + tr * D + c + e) = (f4){y[e], y[e + 1], y[e + 2], y[e + 3]};
                if (c == 0) {
                    part[MT * D + tr] = top;
                    part[MT * D + MT + tr] = sum;
                }
            }
        }
        __syncthreads();
        if (begins && !last_part) {
            cut.more = (int)((w.units - run.count + run.quota - 1) / run.quota);
            cut.kvh = run.kvh;
            cut.first = w.first;
            cut.rows = w.rows;
            cut.r0 = w.r0;
        }
        run.count -= min(w.units - run.unit, run.count);
        run.unit = 0;
        if (run.count > 0) next_tile<MT>(p, run);
    }
    if (t == 0) ((Cut*)p.ws)[block] = cut;
}

// Tiles of 128 rows, as tiles_kernel of 16-bit caches (paged_attention.hip), whose tile layouts, step order and masks these are: 32 rows to each of four waves
// that share 32-key tiles of K and V in LDS, there as fp16 codes. What differs:
//
// * A tile's codes are copied to LDS as they are, widened once for all four waves, 16 (D = 64: 8) a thread of K and of V, and written to the stage two tiles ahead. A
//   wave's eight rows of a tile lie in one page.
// * Keys 0-15 and 16-31 of a tile have a scale each, and are the two halves in which P is made: the scale of K (times the row's factor) is the factor of the
//   exponent's product anyway, and the scale of V, relative to the row's vm, goes into the exponent as its logarithm. l then gets a half's sum of
//   rounded P times what takes that out again. So full steps do nothing more per score than those of a 16-bit cache.
// * Where a scale of V is above the row's vm, or below it by more than 2^8, or is not finite, the step is not a full one: the plain steps sum P before it
//   is scaled, and move vm (to twice the scale: O is then seldom rescaled).
//
// A chunk of 2048 tokens over 14336 keys, 32 heads over 8 of 128: 612 us and 15 of the merge in a kernel trace of 400 calls once the clock has settled (695 in the first 40,
// up to 830 from an idle GPU), whole calls 615 to 640 by the box, 0.80 to 0.83 PFLOP/s, 62 to 64% of a library product of 8192^3. The 16-bit cache takes 564 over normal values, 604 over those
// that these codes stand for. Products take 37% of the cycles and vector work 56% (ten instructions a product, where the 16-bit kernel has five: widening, scales), which add up on a SIMD. Two workgroups a CU: at three the registers
// spill (1920 us). Widening at the start of a step 655, beside the products and two tiles ahead 619; V read ahead of the look at P no faster. With D = 64, half the
// products beside the same vector work, 414 (16-bit: 312).
#define TILES8_WGS(D, MOD) ((D) == 64 && !(MOD) ? 3 : 2)
#define LIFT_TILES 9.f        // P stands 2^9 vs / vm above 2^(x - m), of which at most 2^2 are in a plain step
#define MOST_TILES 32768.f    // of a full step's sum of P in a lane, so that no P is above it
#define LEAST_RATIO -8.f      // log2 of vs / vm

template <int D>
struct Tiles8Lds {
    using L = TilesLds<D>;
    static constexpr int RAW = (L::BYTES + 255) / 256 * 256, HALF = 32 * D, BYTES = RAW + 4 * HALF;  // codes of two tiles, K and V of each
};

template <class T, int D, bool MOD>
__global__ __launch_bounds__(256, TILES8_WGS(D, MOD)) void tiles8_kernel(Attn8Args p) {
    constexpr int MT = 128, UK = 32, AHEAD = ahead(MT, MOD), ROW = 2 * D, KS = D / 16, DT = D / 32;
    constexpr int CB = D / 8;  // codes of a thread
    constexpr int CR = 1024 / ROW;  // rows of a store of the output
    using L = TilesLds<D>;
    typedef typename std::conditional<D == 128, u4v, u2v>::type raw_t;
    typedef __attribute__((address_space(1))) float global_float_t;  // (flat loads would count as LDS accesses too)
    extern __shared__ __attribute__((aligned(256))) char smem[];
    const int lane = threadIdx.x & 63, g = lane >> 5, lq = lane & 31;
    const int wave = uniform((int)(threadIdx.x >> 6));
    const int block = work_block(p.grid);
    Run run = find_run<MT, UK, AHEAD, 256, true>(p, (int*)smem, (u32*)(smem + L::SHARED), block);
    Cut cut = {};
    const u32 smem_u = lds_addr(smem);

    while (run.count > 0) {
        const WorkTile w = uniform(make_tile<MT, UK, AHEAD, true>(p, run.b, run.j));
        if (run.unit + run.count <= AHEAD) break;  // the next run's
        const bool begins = run.unit == 0, last_part = run.unit + run.count >= w.units, whole = begins && last_part;
        const int u0 = begins ? 0 : run.unit - AHEAD, u1 = min(w.units, run.unit + run.count) - AHEAD, n = w.hi > w.lo ? u1 - u0 : 0;
        const int* table = p.table + run.b * p.pitch;
        const signed char* kbase = uniform((const signed char*)p.k + run.kvh * p.kph);
        const signed char* vbase = uniform((const signed char*)p.v + run.kvh * p.vph);
        const float *ksbase = uniform(p.ks + run.kvh * p.ksh), *vsbase = uniform(p.vs + run.kvh * p.vsh);
        const int key_first = w.lo + u0 * UK, last16 = (w.hi - 1) & ~15, head = w.head - u0;  // key_first: were no keys skipped
        auto key_of = [&](int i) __attribute__((always_inline)) { return key_first + i * UK + (i >= head ? w.skip : 0); };
        const int wr0 = w.r0 + 32 * wave;  // the wave's first row
        const bool active = wr0 <= w.r1;
        const int n0 = uniform(w.p0 + div_by(min(wr0, w.r1), p.G)), n1 = uniform(w.p0 + div_by(min(wr0 + 31, w.r1), p.G));

        // What the tiles from `base` on need, tile base + lane in a lane, read anew every ~58 of them: the page of the wave's rows, and of keys 0-15 and 16-31 the
        // scale of K (NaN if it is not finite), log2 of that of V, and its reciprocal.
        int base = 0, ids = 0;
        float ks0 = 0.f, ks1 = 0.f, lv0 = 0.f, lv1 = 0.f, iv0 = 0.f, iv1 = 0.f;
        bool hole = false;  // whether the cache lacks a page of the lane's tile
        auto look_up = [&](int from) __attribute__((always_inline)) {  // the pages, and the scales' loads (of V into lv0 and lv1)
            base = from;
            const int key = key_of(min(from + lane_again(), n - 1)), k0 = min(key, last16), k1 = min(key + 16, last16), e0 = div_by(k0, p.S), e1 = div_by(k1, p.S);
            const u32 t0 = (u32)table[e0], t1 = (u32)table[e1], p0 = t0 < (u32)p.P ? t0 : 0, p1 = t1 < (u32)p.P ? t1 : 0;
            const u32 r0 = (u32)(k0 - e0 * (int)p.S.d) >> p.shift, r1 = (u32)(k1 - e1 * (int)p.S.d) >> p.shift;
            hole = p0 != t0 || p1 != t1;
            ids = (int)(wave >> 1 ? p1 : p0);
            ks0 = *(const global_float_t*)(ksbase + row_at(p0, p.ksp, r0, p.ksb));
            ks1 = *(const global_float_t*)(ksbase + row_at(p1, p.ksp, r1, p.ksb));
            lv0 = *(const global_float_t*)(vsbase + row_at(p0, p.vsp, r0, p.vsb));
            lv1 = *(const global_float_t*)(vsbase + row_at(p1, p.vsp, r1, p.vsb));
        };
        auto make_scales = [&]() __attribute__((always_inline)) {
            ks0 = ks0 <= FLT_TOP ? ks0 : __builtin_nanf("");
            ks1 = ks1 <= FLT_TOP ? ks1 : __builtin_nanf("");
            iv0 = __builtin_amdgcn_rcpf(lv0);
            iv1 = __builtin_amdgcn_rcpf(lv1);
            lv0 = __builtin_amdgcn_logf(lv0);
            lv1 = __builtin_amdgcn_logf(lv1);
        };
        auto refresh = [&](int from) __attribute__((always_inline)) {
            look_up(from);
            make_scales();
        };
        auto of_tile = [&](float x, int i) __attribute__((always_inline)) { return __int_as_float(__builtin_amdgcn_readlane(__float_as_int(x), i - base)); };

        // Codes come by direct copies, two tiles ahead of where they are widened: the wave's rows 8 wave .. + 7 of tile t to the half t % 2 of RAW, 16 bytes a lane
        // (D = 64: of half the lanes), and each thread widens 16 (8) of its own wave's codes for the stages that all four read. Rows behind the sequence's end in
        // its last 16 keys are read as they are, later ones as those 16. Past the run's last tile that one is copied again, so that there are always two copies
        // behind those that are waited for.
        using LDS = Tiles8Lds<D>;
        constexpr int LANES = D / 16;  // of a row
        const u32 k_off = (u32)(lane / LANES) * p.kpr + (lane % LANES) * 16, v_off = (u32)(lane / LANES) * p.vpr + (lane % LANES) * 16;
        auto issue = [&](int t) __attribute__((always_inline)) {
            const int tile = min(t, n - 1), key = min(key_of(tile) + 16 * (wave >> 1), last16), row = key - div_by(key, p.S) * (int)p.S.d + 8 * (wave & 1);
            const u32 page = (u32)__builtin_amdgcn_readlane(ids, tile - base);
            const signed char *k = uniform(kbase + row_at(page, p.kpp, (u32)row, p.kpr)), *v = uniform(vbase + row_at(page, p.vpp, (u32)row, p.vpr));
            const char* to = smem + LDS::RAW + (t & 1) * 2 * LDS::HALF + wave * (8 * D);
            if (D == 128 || lane_again() < 32) {
                dma16(k, k_off, to);
                dma16(v, v_off, to + LDS::HALF);
            }
        };
        const int my_row = 8 * wave + (lane >> 3);
        u32 k_to = (u32)(my_row * ROW + (((lane & 7) * (CB / 8) ^ (D == 128 ? my_row & 15 : my_row >> 1 & 7)) << 4));
        u32 v_to = (u32)(L::V + my_row * ROW + (((lane & 7) * (CB / 8) ^ (D == 128 ? (my_row & 3) << 2 : (my_row >> 1 & 1) << 2)) << 4));
        auto raw_of = [&](int t, int half) __attribute__((always_inline)) {
            return *(const raw_t*)(smem + LDS::RAW + (t & 1) * 2 * LDS::HALF + half * LDS::HALF + wave * (8 * D) + lane_again() * CB);
        };
        // Chunk c of 16 bytes in the stages: half h of it, the second one with the store of both. The two chunks of a thread differ by the last bit of their place.
        u2v wide;
        auto put_half = [&](const raw_t& raw, int c, int h, u32 to) __attribute__((always_inline)) {
            const u2v x = widen4(raw[2 * c + h]);
            if (h == 0) wide = x;
            else *(u4v*)(smem + (to ^ (u32)(c << 4))) = (u4v){wide[0], wide[1], x[0], x[1]};
        };
        // Step i's part: tile i + 2 to its stage, tile i + 4's copies.
        auto advance = [&](int i, u32 st2) __attribute__((always_inline)) {
            if (i + 5 - base > 63) refresh(i);
            wait_copies_but<2>();
            if (i + 2 < n) {
                const raw_t k = raw_of(i + 2, 0), v = raw_of(i + 2, 1);
#pragma unroll
                for (int x = 0; x < CB / 4; x++) put_half(k, x / 2, x % 2, st2 + k_to);
#pragma unroll
                for (int x = 0; x < CB / 4; x++) put_half(v, x / 2, x % 2, st2 + v_to);
            }
            issue(i + 4);
        };
        // A run's start is a chain of accesses to memory: Q goes out first, then table entries, then scales and the first copies together (2 x 4096 rows capped in a window of 2048:
        // 222.5 -> 219.5 us). Q as the B operand of S^T = K Q^T: fp16, its row's largest brought to 2^14 to 2^15, which `by` takes back.
        u4v qf[KS];
        float slope = 0.f, by = 0.f;
        int pos = 0;
        if (active) {
            const int row = min(wr0 + lq, w.r1), token = div_by(row, p.G), head = run.kvh * (int)p.G.d + row - token * (int)p.G.d;
            const T* src = (const T*)p.q + (long)(w.first + token) * p.sqt + head * p.sqh;
#pragma unroll
            for (int x = 0; x < KS; x++) qf[x] = *(const u4v*)(src + (2 * x + g) * 8);
            if constexpr (MOD) {
                if (p.slopes) slope = p.slopes[head] * LOG2E;
                pos = w.p0 + token;
            }
        }
        if (n > 0) {
            look_up(0);
            issue(0);
            issue(1);
        }
        if (active) {
            float top = 0.f;
            auto values = [&](int x) __attribute__((always_inline)) {
                typedef T t8 __attribute__((ext_vector_type(8)));
                return __builtin_convertvector(__builtin_bit_cast(t8, qf[x]), f8);
            };
#pragma unroll
            for (int x = 0; x < KS; x++) {
                const f8 v = values(x);
#pragma unroll
                for (int e = 0; e < 8; e++) top = fmaxf(top, fabsf(v[e]));
            }
            const f2 h = both_halves(top);
            top = fmaxf(h[0], h[1]);
            const int up = top > 0.f && top <= FLT_TOP ? 15 - __builtin_amdgcn_frexp_expf(top) : 0;
            by = ldexpf(p.scale, -up);
#pragma unroll
            for (int x = 0; x < KS; x++) {
                f8 v = values(x);
#pragma unroll
                for (int e = 0; e < 8; e++) v[e] = ldexpf(v[e], up);
                qf[x] = __builtin_bit_cast(u4v, __builtin_convertvector(v, h8));
            }
#pragma unroll
            for (int x = 0; x < KS; x++) asm volatile("" : "+v"(qf[x]));  // made here, not inside the tile loop
        }
        bool holes = false;  // whether the cache lacks any page of the run's part
        if (n > 0) {
            make_scales();
            holes = __any(hole);
            wait_copies();
#pragma unroll
            for (int t = 0; t < 2; t++) {
                const raw_t k = raw_of(t, 0), v = raw_of(t, 1);
#pragma unroll
                for (int x = 0; x < CB / 4; x++) put_half(k, x / 2, x % 2, t * L::TILE + k_to);
#pragma unroll
                for (int x = 0; x < CB / 4; x++) put_half(v, x / 2, x % 2, t * L::TILE + v_to);
            }
            issue(2);
            issue(3);
            if (n > 64) {  // more tiles than the lanes looked at
                const int e1 = div_by(min(key_of(n - 1) + UK, w.hi) - 1, p.S);  // (with what is skipped)
                bool any = false;
                for (int e = div_by(key_of(0), p.S) + lane_again(); e <= e1; e += 64) any |= (u32)table[e] >= (u32)p.P;
                holes = __any(any);
            }
        }

        f16v o[DT];
#pragma unroll
        for (int d = 0; d < DT; d++) o[d] = (f16v){};
        float m = LEAST, l = 0.f, l_old = 0.f, vm = 1e-35f, lvm = -116.26748f;  // lvm: log2 of vm; 512 / vm stays finite

        if (!active) {  // no rows: the wave copies its part
            if (n > 0) __syncthreads();
            u32 st2 = 2 * L::TILE;
            for (int i = 0; i < n; i++) {
                advance(i, st2);
                st2 = st2 == 2 * L::TILE ? 0 : st2 + L::TILE;
                __syncthreads();
            }
        } else {
            // The lane's K reads: row lq, chunk 2 x + g, at k_base ^ 32 x. Its V^T reads: lane i of 16 reads 8 bytes of row 4 g + i / 4 and gets the
            // transposed values; chunk 4 d on of the row at v_base ^ 64 d.
            u32 k_base = smem_u + (u32)(lq * ROW + ((g ^ (D == 128 ? lq & 15 : lq >> 1 & 7)) << 4));
            u32 v_base;
            {
                const int sg = lane & 15, vr = 4 * g + (sg >> 2), c = 2 * (lane >> 4 & 1) + (sg >> 1 & 1);
                v_base = smem_u + (u32)(L::V + vr * ROW + (sg & 1) * 8 + ((c ^ (D == 128 ? (vr & 3) << 2 : (vr >> 1 & 1) << 2)) << 4));
            }
            asm volatile("" : "+v"(k_base), "+v"(v_base));

            // `st`: the offset of the tile's stage (the xors above leave a stage's bits alone).
            auto qk = [&](u32 st, float (&out)[16], auto&& hook) __attribute__((always_inline)) {
                u32 kb = k_base + st;
                asm volatile("" : "+v"(kb));
                f16v acc = {};
                u4v ka[KS / 2];
#pragma unroll
                for (int x = 0; x < KS / 2; x++) ka[x] = lds_u4(kb ^ (u32)(32 * x));
                __builtin_amdgcn_sched_barrier(0);
                __builtin_amdgcn_s_setprio(1);
                __builtin_amdgcn_sched_barrier(0);
#pragma unroll
                for (int x = 0; x < KS; x++) {
                    acc = product32<half_t>(ka[x % (KS / 2)], qf[x], acc);
                    if (x < KS / 2) ka[x] = lds_u4(kb ^ (u32)(32 * (KS / 2 + x)));
                    hook(x);
                    __builtin_amdgcn_sched_barrier(0);
                }
                __builtin_amdgcn_s_setprio(0);
                __builtin_amdgcn_sched_barrier(0);
#pragma unroll
                for (int r = 0; r < 16; r++) out[r] = acc[r];
            };
            // The keys of a tile that the lane's row sees, a bit each.
            auto seen_keys = [&](int key0) __attribute__((always_inline)) {
                auto below = [&](int key) __attribute__((always_inline)) { return (u32)((1ull << min(max(key - key0, 0), 32)) - 1); };
                const int ln = lane_again(), at = w.p0 + div_by(min(wr0 + (ln & 31), w.r1), p.G);
                u32 seen = below(min(at + 1, w.hi));
                if (p.window > 0) seen &= ~below(at - p.window + 1);
                seen |= below(w.prefix);  // at most hi
                if (holes) {
                    const int key = min(key0 + (ln & 31), w.hi - 1);
                    seen &= (u32)__ballot((u32)table[div_by(key, p.S)] < (u32)p.P);
                }
                return seen;
            };
            // What x is times in the softmax's exponent, besides the scales: capped scores without a bias stay the -1 / (1 + 2^e) of their tanh (see capped), times
            // 2 cap. (From HIGH_CAP on, 2 cap passes 4096 and they are made whole first, as large scores are, below.)
            const float scale = MOD && p.cap > 0.f && !p.slopes && p.cap < HIGH_CAP ? 2.f * p.cap : 1.f;
            // Changed scores: c0, c1 the factors of the two halves' products.
            auto bias = [&](float (&x)[16], int key0, float c0, float c1) __attribute__((always_inline)) {
                if constexpr (MOD) {
#pragma unroll
                    for (int r = 0; r < 16; r++) x[r] *= r < 8 ? c0 : c1;
                    if (__builtin_expect(p.cap >= HIGH_CAP, 0)) {
#pragma unroll
                        for (int r = 0; r < 16; r++) x[r] = capped<true>(x[r], p.cap);
                    } else if (p.cap > 0.f) {
#pragma unroll
                        for (int r = 0; r < 16; r++) x[r] = __builtin_amdgcn_rcpf(-1.f - __builtin_amdgcn_exp2f(x[r]));
                        if (scale != 1.f) return;
#pragma unroll
                        for (int r = 0; r < 16; r++) x[r] = __builtin_fmaf(2.f * p.cap, x[r], p.cap);
                    }
                    if (p.slopes) {
                        const float d0 = (float)(pos - key0 - 4 * g);
#pragma unroll
                        for (int r = 0; r < 16; r++) x[r] = __builtin_fmaf(-slope, fabsf(d0 - (float)(8 * (r >> 2) + (r & 3))), x[r]);
                    }
                }
            };
            u4v pf[2];  // P of the two 16-key halves
            // The tile at hand in full steps: of half h, 2^(fma(x, factor, add)) is P; sum of P so far; what takes P's scale out of a sum.
            float factor1 = 1.f, add1 = 0.f, sum0 = 0.f, sum1 = 0.f, back0 = 0.f, back1 = 0.f;
            // Part k (of four) of a half's P.
            auto exps = [&](const float* x, int k, u4v& d, float factor, float add, float& sum) __attribute__((always_inline)) {
                const float a = __builtin_amdgcn_exp2f(__builtin_fmaf(x[2 * k], factor, add)), b = __builtin_amdgcn_exp2f(__builtin_fmaf(x[2 * k + 1], factor, add));
                const u32 word = pair_of<half_t>(a, b);
                sum = add_pair<half_t>(word, sum);
                d[k] = word;
            };
            // A half's P of a plain step: scores are whole, P is summed first, then times f.
            auto exps_plain = [&](const float* x, u4v& d, float f) __attribute__((always_inline)) {
#pragma unroll
                for (int k = 0; k < 4; k++) {
                    const float a = __builtin_amdgcn_exp2f(x[2 * k] - m), b = __builtin_amdgcn_exp2f(x[2 * k + 1] - m);
                    l += a;
                    l += b;
                    d[k] = pair_of<half_t>(a * f, b * f);
                }
            };
            auto no_hook = [](int) {};
            auto read_v = [&](u32 vb, int j, int d) __attribute__((always_inline)) {
                const u32 at = (vb ^ (u32)(64 * d)) + 16 * j * ROW;
                return __builtin_shufflevector(lds_tr(at), lds_tr(at + 8 * ROW), 0, 1, 2, 3);
            };
            auto pv = [&](u32 st, auto&& hook) __attribute__((always_inline)) {
                u32 vb = v_base + st;
                asm volatile("" : "+v"(vb));
                u4v va[DT];
#pragma unroll
                for (int d = 0; d < DT; d++) va[d] = read_v(vb, 0, d);
                __builtin_amdgcn_sched_barrier(0);
#pragma unroll
                for (int d = 0; d < DT; d++) {
                    o[d] = product32<half_t>(va[d], pf[0], o[d]);
                    va[d] = read_v(vb, 1, d);
                    hook(d);
                    __builtin_amdgcn_sched_barrier(0);
                }
#pragma unroll
                for (int d = 0; d < DT; d++) {
                    o[d] = product32<half_t>(va[d], pf[1], o[d]);
                    hook(DT + d);
                    __builtin_amdgcn_sched_barrier(0);
                }
            };

            // Tiles all of whose keys all of the wave's rows see: full0 .. full1 - 1.
            int full0 = 0, full1 = 0;
            float sa[16], sb[16];
            bool large = false;
            // A tile's first part, wherever it lies: its scores, whole (x factor - m in one rounding would leave fp32's range where scores pass 2^24: a wave that
            // meets one of 4096 or more takes no full steps from then on), masked where not every row sees every key, the maximum, vm, and the first half of P.
            // Returns whether full steps may follow; half1: what the second half's P is times.
            auto begin_tile = [&](int i, u32 st, u32 seen, bool masked, float& half1) __attribute__((always_inline)) {
                qk(st, sa, no_hook);
                const float c0 = by * of_tile(ks0, i), c1 = by * of_tile(ks1, i), vs0 = __builtin_amdgcn_rcpf(of_tile(iv0, i)), vs1 = __builtin_amdgcn_rcpf(of_tile(iv1, i));
                if constexpr (MOD) bias(sa, key_of(i), c0, c1);
#pragma unroll
                for (int r = 0; r < 16; r++) sa[r] *= MOD ? scale : r < 8 ? c0 : c1;
                if constexpr (!MOD) {
                    if (!large) {
                        float a = 0.f;
#pragma unroll
                        for (int r = 0; r < 16; r++) a = fmaxf(a, fabsf(sa[r]));
                        large = __any(a >= 4096.f);
                    }
                }
                if (masked) {
                    const u32 mine = seen >> (4 * (lane_again() >> 5));  // register r: key 8 (r / 4) + 4 g + r % 4
#pragma unroll
                    for (int r = 0; r < 16; r++) sa[r] = mine >> (8 * (r >> 2) + (r & 3)) & 1 ? sa[r] : -__builtin_inff();
                }
                float mx = sa[0];
#pragma unroll
                for (int r = 1; r < 16; r++) mx = fmaxf(mx, sa[r]);
                const f2 h = both_halves(mx);
                mx = fmaxf(h[0], h[1]);
                const bool see0 = seen & 0xffffu, see1 = seen >> 16;
                const float v0 = see0 && vs0 <= FLT_TOP ? vs0 : 0.f, v1 = see1 && vs1 <= FLT_TOP ? vs1 : 0.f, vx = fmaxf(v0, v1);
                if (__any(mx > m + 2.f || vx > vm)) {
                    const float mn = mx > m + 2.f ? mx : m, vn = vx > vm ? fminf(2.f * vx, FLT_TOP) : vm, a = __builtin_amdgcn_exp2f(m - mn);
                    const float b = a * (vm / vn);
                    m = mn;
                    vm = vn;
                    lvm = __builtin_amdgcn_logf(vn);
                    l *= a;
#pragma unroll
                    for (int d = 0; d < DT; d++) o[d] *= b;
                }
                l_old = l;
                if ((see0 && !(vs0 <= FLT_TOP)) || (see1 && !(vs1 <= FLT_TOP))) l = l_old = __builtin_nanf("");
                const float unit = 512.f / vm;
                half1 = v1 * unit;
                exps_plain(sa, pf[0], v0 * unit);
                // For a full step that follows: the scores are whole, P's first half is in l.
                sum0 = 0.f;
                back0 = 0.f;
                factor1 = 1.f;
                const float d1 = of_tile(lv1, i) - lvm + LIFT_TILES;
                add1 = d1 - m;
                back1 = vm * (1.f / 512.f) * of_tile(iv1, i);
                return !large && !__any(!(d1 <= LIFT_TILES && d1 >= LIFT_TILES + LEAST_RATIO));
            };
            // A step of the full tiles: tile i's scores are in s, its P's first half in pf[0] and sum0 (or in l); tile i + 1 is full
            // too, and its scores go to nxt. Steps of KS (or 2 DT = KS) products: the four parts of half a tile's exponentials beside every
            // (KS / 4)-th. P is made with the m and vm at hand: a lane's sum of no more than MOST_TILES proves that no P was above it; else, or where tile i + 1's
            // scales of V do not suit vm, the step ends before the product (false), and the tile is taken again by a plain step.
            auto beside = [](int x) __attribute__((always_inline)) { return x % (KS / 4) == KS / 4 - 1; };
            auto full_step = [&](int i, u32 st, u32 st1, u32 st2, const float (&s)[16], float (&nxt)[16]) __attribute__((always_inline)) {
                // Tile i + 2 (there is one) goes to its stage beside the products, half a chunk beside every second one: their vector work and the products overlap.
                wait_copies_but<2>();
                const raw_t now_k = raw_of(i + 2, 0);
                auto put_beside = [&](const raw_t& raw, int x, u32 to) __attribute__((always_inline)) {
                    if (x % 2 == 0 && x / 2 < CB / 4) put_half(raw, x / 4, x / 2 & 1, to);
                };
                sum1 = 0.f;
                qk(st1, nxt, [&](int x) {
                    if (beside(x)) exps(s + 8, x / (KS / 4), pf[1], factor1, add1, sum1);
                    put_beside(now_k, x, st2 + k_to);
                });
                const raw_t now_v = raw_of(i + 2, 1);
                const float d0 = of_tile(lv0, i + 1) - lvm, d1 = of_tile(lv1, i + 1) - lvm;
                if (__builtin_expect(__any(!(sum0 + sum1 <= MOST_TILES && fmaxf(d0, d1) <= 0.f && d0 >= LEAST_RATIO && d1 >= LEAST_RATIO)), 0)) {
#pragma unroll
                    for (int x = 0; x < CB / 4; x++) put_half(now_v, x / 2, x % 2, st2 + v_to);
                    issue(i + 4);
                    return false;
                }
                const float c0 = by * of_tile(ks0, i + 1), c1 = by * of_tile(ks1, i + 1);
                bias(nxt, key_of(i + 1), c0, c1);
                l = __builtin_fmaf(sum0, back0, __builtin_fmaf(sum1, back1, l));
                l_old = l;
                const float factor0 = MOD ? scale : c0, add0 = d0 + LIFT_TILES - m, unit = vm * (1.f / 512.f);
                factor1 = MOD ? scale : c1;
                add1 = d1 + LIFT_TILES - m;
                back0 = unit * of_tile(iv0, i + 1);
                back1 = unit * of_tile(iv1, i + 1);
                sum0 = 0.f;
                u4v pn;
                pv(st, [&](int x) {
                    if (beside(x)) {
                        exps(nxt, x / (KS / 4), pn, factor0, add0, sum0);
                        asm volatile("" : "+v"(pn), "+v"(sum0));
                    }
                    put_beside(now_v, x, st2 + v_to);
                });
                pf[0] = pn;
                issue(i + 4);
                __syncthreads();
                return true;
            };

            if (n > 0) {
                __syncthreads();
                if (!holes) {
                    const int upto = min(w.hi, p.window > 0 ? n0 + 1 : max(n0 + 1, w.prefix));
                    const int window_first = key_first + w.skip;
                    full0 = first_unit_in_window<UK>(n1, p.window, window_first);
                    if (w.skip) full0 = max(full0, head);
                    full1 = min(max((upto - window_first) / UK, 0), n);
                }
            }
            const int last = full1 - 3;  // pairs of full steps i, i + 1 up to it: tiles .. i + 2 are full
            u32 st = 0, st1 = L::TILE, st2 = 2 * L::TILE;  // the stages of tiles i, i + 1, i + 2
            auto turn_stages = [&]() __attribute__((always_inline)) {
                const u32 x = st;
                st = st1;
                st1 = st2;
                st2 = x;
            };
            for (int i = 0; i < n;) {
                const bool masked = i < full0 || i >= full1;
                u32 seen = ~0u;
                if (masked) seen = seen_keys(key_of(i));
                bool full = i >= full0 && i <= last, copied = false;  // whether step i's part of the copies is done
                if (!full) {
                    advance(i, st2);
                    copied = true;
                }
                if (__any(seen != 0)) {
                    float half1;
                    while (true) {
                        const bool may = begin_tile(i, st, seen, masked, half1);
                        full = full && may;
                        bool done = true, taken = true;  // taken: the tile's maximum is
                        while (full) {
                            if (i + 6 - base > 63) refresh(i);
                            taken = false;
                            done = full_step(i, st, st1, st2, sa, sb);
                            if (!done) break;
                            i++;
                            turn_stages();
                            done = full_step(i, st, st1, st2, sb, sa);
                            if (!done) break;
                            i++;
                            turn_stages();
                            full = i <= last;
                        }
                        if (done) {
                            if (!copied) advance(i, st2);
                            copied = true;
                            if (taken) {
                                exps_plain(sa + 8, pf[1], half1);
                                break;
                            }
                            sum1 = 0.f;
#pragma unroll
                            for (int k = 0; k < 4; k++) exps(sa + 8, k, pf[1], factor1, add1, sum1);
                            if (!__any(!(sum0 + sum1 <= MOST_TILES))) {
                                l = __builtin_fmaf(sum0, back0, __builtin_fmaf(sum1, back1, l));
                                break;
                            }
                        }
                        // P above the maximum at hand, or a scale of V that does not suit: the tile again by a plain step, its copies made.
                        l = l_old;
                        copied = true;
                        full = false;
                    }
                    pv(st, no_hook);
                }
                i++;
                turn_stages();
                __syncthreads();
            }
        }

        wait_copies();  // those behind the last tile
        // The rows turn around in LDS (chunk c of row r at c ^ (r & 15) or, of 8, c ^ (r & 7)) so that a store covers whole rows.
        if (active) {
            const int ln = lane_again(), lg = ln >> 5, lr = ln & 31;
            const f2 lh = both_halves(l);
            const float sum = lh[0] + lh[1], unit = vm * (1.f / 512.f);
            char* turn = smem + wave * (32 * 256);
            auto settle_lds = []() __attribute__((always_inline)) {
                __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
                __builtin_amdgcn_wave_barrier();
                __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
            };
            if (whole) {
                const float inv = sum == 0.f ? 0.f : 1.f / sum;  // a row that saw nothing: O is 0
#pragma unroll
                for (int d = 0; d < DT; d++)
#pragma unroll
                    for (int r4 = 0; r4 < 4; r4++) {
                        const f4 y = (f4){o[d][4 * r4], o[d][4 * r4 + 1], o[d][4 * r4 + 2], o[d][4 * r4 + 3]} * unit * inv;
                        const u2v word = {pair_of<T>(y[0], y[1]), pair_of<T>(y[2], y[3])};
                        *(u2v*)(turn + lr * ROW + (((4 * d + r4) ^ (lr & (D / 8 - 1))) << 4) + 8 * lg) = word;
                    }
                settle_lds();
#pragma unroll
                for (int i = 0; i < 32 / CR; i++) {
                    const int r = CR * i + ln / (D / 8), c = ln % (D / 8), out_row = wr0 + r;
                    const u4v x = *(const u4v*)(turn + r * ROW + ((c ^ (r & (D / 8 - 1))) << 4));
                    if (out_row <= w.r1) {
                        const int token = div_by(out_row, p.G), head = run.kvh * (int)p.G.d + out_row - token * (int)p.G.d;
                        *(u4v*)((T*)p.o + (long)(w.first + token) * p.sot + head * p.soh + c * 8) = x;
                    }
                }
            } else {
                float* part = partial<MT, D>(p, block, begins);
#pragma unroll
                for (int half = 0; half < D / 64; half++) {  // 64 values of fp32 at a time
#pragma unroll
                    for (int d = 0; d < 2; d++)
#pragma unroll
                        for (int r4 = 0; r4 < 4; r4++) {
                            const f16v& z = o[2 * half + d];
                            *(f4*)(turn + lr * 256 + (((8 * d + 2 * r4 + lg) ^ (lr & 15)) << 4)) = (f4){z[4 * r4], z[4 * r4 + 1], z[4 * r4 + 2], z[4 * r4 + 3]} * unit;
                        }
                    settle_lds();
#pragma unroll
                    for (int i = 0; i < 8; i++) {
                        const int r = 4 * i + (ln >> 4), c = ln & 15;
                        *(f4*)(part + (32 * wave + r) * D + 64 * half + 4 * c) = *(const f4*)(turn + r * 256 + ((c ^ (r & 15)) << 4));
                    }
                    settle_lds();
                }
                if (lg == 0) {
                    part[MT * D + 32 * wave + lr] = m;
                    part[MT * D + MT + 32 * wave + lr] = sum;
                }
            }
        }
        __syncthreads();
        if (begins && !last_part) {
            cut.more = (int)((w.units - run.count + run.quota - 1) / run.quota);
            cut.kvh = run.kvh;
            cut.first = w.first;
            cut.rows = w.rows;
            cut.r0 = w.r0;
        }
        run.count -= min(w.units - run.unit, run.count);
        run.unit = 0;
        if (run.count > 0) next_tile<MT>(p, run);
    }
    if (threadIdx.x == 0) ((Cut*)p.ws)[block] = cut;
}

template <class T, int D, int MT>
__global__ __launch_bounds__(256) void merge8_kernel(Attn8Args p) { merge_parts<T, D, MT>(p); }

// ------------------------------------------------------------------------------------------------ launches

struct Plan8 {
    int mt, grid;
    bool spread;
    size_t workspace;
};
static int make_plan8(long T, long B, long H, long Hkv, long D, int type, Plan8* plan) {
    if (T <= 0 || B <= 0 || B > MAX_SEQUENCES || Hkv <= 0 || H <= 0 || H % Hkv || (D != 64 && D != 128) || type < RDA_FP16 || type > RDA_BF16) return RDA_ERR_INVALID;
    if (T * (H / Hkv) >= 1L << 31) return RDA_ERR_INVALID;
    const long rows = T * (H / Hkv) / B;
    // Rows of a tile, by a sequence's mean (a call cannot look at starts): us at tiles of 16 / 32 / 128, D = 128, 32 heads over 8. 32 sequences over 4096 keys of 4 rows 50 / 55 / 76, 16 rows
    // 52 / 57 / 78, 20 rows 61 / 58 / 79, 64 rows 114 / 85 / 98, 96 rows 167 / 144 / 108; one prompt over 2000 of 640 rows 38 / 33 / 39, of 1024 47 / 44 / 41, of 2048 81 / 68 / 52. Both bounds stand
    // where the 16-bit cache's do. What that costs: 8 sequences of 96 rows 55 / 48 / 61 and one of 644 38 / 32 / 42 (128 is taken), and with D = 64 small batches of up to 512 rows, which tiles
    // of 16 take 5 to 15% faster (one prompt of 512 rows 22.4 / 24.9 / 32.9, 32 sequences of 20 rows 40 / 45 / 56; but of 48 rows 73 / 66 / 66).
    plan->mt = rows <= 16 ? 16 : rows <= 64 || B * ((rows + 127) / 128) * Hkv <= 40 ? 32 : 128;
    // Where a sequence's rows of a KV head are one tile no keys are read twice, and runs go to the XCDs in turn, so that each has parts of all heads: a key's codes of
    // a head are 64 or 128 bytes of a row of all heads (in pages laid out token by token), and XCDs of a head each would use few of their caches'
    // channels and read halves of lines twice. 64 sequences over 8192 keys 218 -> 206 us, D = 64 159 -> 112, 256 over 1024 130 -> 120; with two tiles of 32 rows
    // 95 -> 104. (In pages of whole heads, as QuantizedCache.empty lays them out, 188 and 103 either way.)
    plan->spread = rows <= plan->mt;
    plan->grid = plan->mt == 128 && D == 64 ? 768 : 512;
    if ((T * (H / Hkv) / plan->mt + 1) * B >= 1L << 31) return RDA_ERR_INVALID;
    plan->workspace = (size_t)plan->grid * sizeof(Cut) + (size_t)plan->grid * 2 * plan->mt * (D + 2) * 4;
    return 0;
}

template <class T, int D, int MB>
static int launch_rows8(const Attn8Args& a, void* stream) {
    constexpr int OP = D + 4;
    const size_t o = 4 * 16 * OP * 4, sums = (size_t)(a.B + 1) * 4, lds = o > sums ? o : sums;
    const auto launch = [&](auto kernel) { hipLaunchKernelGGL(kernel, dim3(a.grid), dim3(256), lds, (hipStream_t)stream, a); };
    a.cap > 0.f || a.slopes ? launch(rows8_kernel<T, D, MB, true>) : launch(rows8_kernel<T, D, MB, false>);
    if (const hipError_t e = hipGetLastError()) return (int)e;
    hipLaunchKernelGGL((merge8_kernel<T, D, 16 * MB>), dim3(a.grid, 4 * MB), dim3(256), 0, (hipStream_t)stream, a);
    return (int)hipGetLastError();
}

template <class X, class Q, int PS>
static int launch_append8(const Append8Args& a, dim3 grid, size_t lds, void* stream) {
    static std::atomic<size_t> done[RDA_MAX_DEVICES];
    if (lds > 32768)  // angles of 64 tokens and more than 64 pairs, or of 32 and 128: up to 64 KB
        if (const int e = ensure_dynamic_lds((const void*)append8_kernel<X, Q, PS>, lds, done)) return e;
    hipLaunchKernelGGL((append8_kernel<X, Q, PS>), grid, dim3(256), lds, (hipStream_t)stream, a);
    return (int)hipGetLastError();
}

template <class T, int D>
static int launch_tiles8(const Attn8Args& a, void* stream) {
    static std::atomic<size_t> done[2][RDA_MAX_DEVICES];
    const bool mod = a.cap > 0.f || a.slopes;
    if (const int e = ensure_dynamic_lds(mod ? (const void*)tiles8_kernel<T, D, true> : (const void*)tiles8_kernel<T, D, false>, Tiles8Lds<D>::BYTES, done[mod])) return e;
    const auto launch = [&](auto kernel) { hipLaunchKernelGGL(kernel, dim3(a.grid), dim3(256), Tiles8Lds<D>::BYTES, (hipStream_t)stream, a); };
    mod ? launch(tiles8_kernel<T, D, true>) : launch(tiles8_kernel<T, D, false>);
    if (const hipError_t e = hipGetLastError()) return (int)e;
    hipLaunchKernelGGL((merge8_kernel<T, D, 128>), dim3(a.grid, 8), dim3(256), 0, (hipStream_t)stream, a);
    return (int)hipGetLastError();
}

// Codes are read and written 8 and 16 at a time.
static bool code_rows(const void* p, const long* strides) {
    for (int i = 0; i < 3; i++)
        if (strides[i] % 16) return false;
    return ((uintptr_t)p & 15) == 0;
}
static bool cache8_ok(long P, long S, long N, long block) {
    return N > 0 && P > 0 && P < 1L << 31 && S > 0 && (block == 16 || block == 32 || block == 64) && S % block == 0 && N <= MAX_KEYS8 / S;
}

extern "C" {

int rda_paged_append_i8(const void* q, const void* k, const void* v, void* q_out, void* k_codes, void* v_codes, float* k_scales, float* v_scales, const int* table,
                        const int* starts, const int* lengths, const double* turns, float factor, int interleaved, const void* q_weight, const void* k_weight,
                        int weight_type, float eps, int type, int q_type, const long* dims, void* stream) {
    const long T = dims[0], H = dims[1], Hkv = dims[2], D = dims[3], R = dims[4], B = dims[5], N = dims[6], P = dims[8], S = dims[9], block = dims[10];
    if (T <= 0 || T > MAX_ROWS || H < 0 || Hkv <= 0 || H + 2 * Hkv > 65535 || !rotary_ok(turns, D, R) || B <= 0 || B > MAX_SEQUENCES || !cache8_ok(P, S, N, block))
        return RDA_ERR_INVALID;
    if (type < RDA_FP16 || type > RDA_FP32 || q_type < RDA_FP16 || q_type > RDA_BF16 || weight_type < RDA_FP16 || weight_type > RDA_FP32) return RDA_ERR_INVALID;
    if (!vector_rows(k, dims + 13, 2, type) || !vector_rows(v, dims + 15, 2, type) || !code_rows(k_codes, dims + 19) || !code_rows(v_codes, dims + 22)) return RDA_ERR_INVALID;
    if (H && (!vector_rows(q, dims + 11, 2, type) || !vector_rows(q_out, dims + 17, 2, q_type))) return RDA_ERR_INVALID;
    if (!vector_rows(q_weight, dims, 0, type) || !vector_rows(k_weight, dims, 0, type) || (H && !q_weight != !k_weight)) return RDA_ERR_INVALID;
    Append8Args a = {{turns, (int)D, (int)R, interleaved & 1, factor, 1.f}, q, k, v, q_out, (signed char*)k_codes, (signed char*)v_codes, k_scales, v_scales, table, starts,
                     lengths, q_weight, k_weight, weight_type, eps, (int)T, (int)H, (int)Hkv, (int)B, (int)N, (int)P, (int)block, 0, make_div((int)S), dims[7],
                     dims[11], dims[12], dims[13], dims[14], dims[15], dims[16], dims[17], dims[18], dims[19], dims[20], dims[21], dims[22], dims[23], dims[24],
                     dims[25], dims[26], dims[27], dims[28], dims[29], dims[30]};
    const long slots = T / block + 2 * B, heads = H + 2 * Hkv, together = 64 / block;
    // Heads of a workgroup: as many as leave 1024 workgroups, so that angles are made for more than one head at a time (16384 tokens at 512 / 1024 / 2048 / 4096:
    // 103 / 100 / 101 / 112 us).
    long slice = (heads * slots / 1024 + together - 1) / together * together;
    if (slice < together) slice = together;
    if (slice > heads) slice = (heads + together - 1) / together * together;
    a.slice = (int)slice;
    const size_t lds = (size_t)block * (R / 2) * 8;
    const dim3 grid((unsigned)slots, (unsigned)((heads + slice - 1) / slice));
    const int rows = 64 / (int)(D / 16);  // of a pass of a wave
    const auto from = [&](auto x) {
        using X = decltype(x);
        const auto to = [&](auto y) {
            using Q = decltype(y);
            // 64 sequences of 1 / 2 / 3 / 5 / 8 tokens: 4.5 / 7.3 / 10.0 / 15.0 / 25.2 us by tokens, 14.4 / 14.3 / 12.7 / 12.9 / 11.7 by blocks; 256 of one 5.4 and 39.7. The mean decides,
            // since a call cannot look at starts, and a chunk among single tokens is written by one wave for each block and slice of heads: 127 tokens beside a chunk of 256 take 71 us (blocks
            // of 64: 137) where the kernel of blocks would take 23 (40), 63 beside a chunk of 190 70 (137) and 16 (27).
            if (T < 4 * B) {
                const int held = rows, slices = (int)((H + held - 1) / held + 2 * ((Hkv + held - 1) / held));
                hipLaunchKernelGGL((append8_few_kernel<X, Q>), dim3((unsigned)T, (unsigned)((slices + 3) / 4)), dim3(256), 0, (hipStream_t)stream, a);
                return (int)hipGetLastError();
            }
            return rows >= 16 ? launch_append8<X, Q, 1>(a, grid, lds, stream) : rows >= 8 ? launch_append8<X, Q, 2>(a, grid, lds, stream) : launch_append8<X, Q, 4>(a, grid, lds, stream);
        };
        return q_type == RDA_FP16 ? to(half_t{}) : to(bf16_t{});
    };
    return type == RDA_FP16 ? from(half_t{}) : type == RDA_BF16 ? from(bf16_t{}) : from(float{});
}

int rda_paged_read_i8(const void* k_codes, const void* v_codes, const float* k_scales, const float* v_scales, const int* table, const int* starts, const int* lengths,
                      void* k_out, void* v_out, int type, const long* dims, void* stream) {
    const long T = dims[0], Hkv = dims[1], D = dims[2], B = dims[3], N = dims[4], P = dims[6], S = dims[7], block = dims[8];
    if (T <= 0 || T > MAX_ROWS || Hkv <= 0 || Hkv > 65535 || D <= 0 || D % 16 || D > 2 * MAX_PAIRS || B <= 0 || B > MAX_SEQUENCES || !cache8_ok(P, S, N, block)) return RDA_ERR_INVALID;
    if (type < RDA_FP16 || type > RDA_FP32 || !code_rows(k_codes, dims + 9) || !code_rows(v_codes, dims + 12) || !vector_rows(k_out, dims, 0, type) ||
        !vector_rows(v_out, dims, 0, type))
        return RDA_ERR_INVALID;
    const Read8Args a = {(const signed char*)k_codes, (const signed char*)v_codes, k_scales, v_scales, table, starts, lengths, k_out, v_out,
                         (int)T, (int)Hkv, (int)D, (int)B, (int)N, (int)P, block == 16 ? 4 : block == 32 ? 5 : 6, make_div((int)S), dims[5],
                         dims[9], dims[10], dims[11], dims[12], dims[13], dims[14], dims[15], dims[16], dims[17], dims[18], dims[19], dims[20]};
    const auto launch = [&](auto kernel) {
        hipLaunchKernelGGL(kernel, dim3((unsigned)((T + 3) / 4)), dim3(256), 0, (hipStream_t)stream, a);
        return (int)hipGetLastError();
    };
    return type == RDA_FP16 ? launch(read8_kernel<half_t>) : type == RDA_BF16 ? launch(read8_kernel<bf16_t>) : launch(read8_kernel<float>);
}

size_t rda_paged_attn_i8_workspace(long T, long B, long H, long Hkv, long D, int type) {
    Plan8 plan;
    return make_plan8(T, B, H, Hkv, D, type, &plan) ? 0 : plan.workspace;
}

int rda_paged_attn_i8(const void* q, void* out, const void* k_codes, const void* v_codes, const float* k_scales, const float* v_scales, const int* table,
                      const int* starts, const int* lengths, const int* prefix, const float* slopes, void* workspace, float scale, float softcap, int window, int fill,
                      int type, const long* dims, void* stream) {
    const long T = dims[0], H = dims[1], Hkv = dims[2], D = dims[3], B = dims[4], N = dims[5], P = dims[7], S = dims[8], block = dims[9];
    Plan8 plan;
    if (const int e = make_plan8(T, B, H, Hkv, D, type, &plan)) return e;
    if (!cache8_ok(P, S, N, block) || window < 0 || !(softcap >= 0.f) || ((uintptr_t)workspace & 15)) return RDA_ERR_INVALID;
    if (!vector_rows(q, dims + 10, 2, type) || !vector_rows(out, dims + 12, 2, type) || !code_rows(k_codes, dims + 14) || !code_rows(v_codes, dims + 17)) return RDA_ERR_INVALID;
    // Units of a KV head in 32 bits, whatever the lengths.
    if ((T * (H / Hkv) / plan.mt + B) * (N * S / 32 + 1 + ahead(plan.mt, false)) >= 1L << 32) return RDA_ERR_INVALID;
    for (int i : {14, 15, 17, 18, 20, 21, 23, 24})
        if (dims[i] < 0 || dims[i] >= (i == 15 || i == 18 ? 1L << 28 : 1L << 32)) return RDA_ERR_INVALID;  // eight rows of codes: 32-bit offsets
    Attn8Args a;
    a.q = q; a.o = out; a.k = k_codes; a.v = v_codes;
    a.ks = k_scales; a.vs = v_scales;
    a.table = table; a.starts = starts; a.lengths = lengths; a.prefix = prefix;
    a.slopes = slopes;
    a.ws = (char*)workspace;
    a.T = (int)T; a.B = (int)B; a.H = (int)H; a.Hkv = (int)Hkv; a.P = (int)P; a.N = (int)N; a.capacity = (int)(N * S);
    a.S = make_div((int)S); a.G = make_div((int)(H / Hkv));
    a.shift = block == 16 ? 4 : block == 32 ? 5 : 6;
    a.pitch = dims[6];
    a.sqt = dims[10]; a.sqh = dims[11]; a.sot = dims[12]; a.soh = dims[13];
    a.kpp = (u32)dims[14]; a.kpr = (u32)dims[15]; a.kph = dims[16]; a.vpp = (u32)dims[17]; a.vpr = (u32)dims[18]; a.vph = dims[19];
    a.ksp = (u32)dims[20]; a.ksb = (u32)dims[21]; a.ksh = dims[22]; a.vsp = (u32)dims[23]; a.vsb = (u32)dims[24]; a.vsh = dims[25];
    a.scale = softcap > 0.f ? scale / softcap * 2.f * LOG2E : scale * LOG2E;
    a.cap = softcap * LOG2E;
    // Normal, positive and finite: masked scores are -inf before they meet the scale.
    if (!(a.scale >= 1.2e-38f && a.scale <= 3e38f && a.cap <= 3e38f)) return RDA_ERR_INVALID;
    a.window = window;
    // No more workgroups than units there can be: a short table of few sequences needs none that finds no work.
    const long least = plan.mt == 128 ? 32 : 128 * rows8_steps(plan.mt / 16), units = (T * (H / Hkv) / plan.mt + B) * ((N * S + least - 1) / least + ahead(plan.mt, false)) * Hkv;
    const int most = softcap > 0.f || slopes ? 512 : plan.grid;
    a.grid = (int)(units < most ? units : most);
    a.runs = make_div(a.grid);
    a.fill = fill;
    a.spread = plan.spread;
    const auto heads = [&](auto x) {
        using X = decltype(x);
        if (plan.mt == 128) return D == 64 ? launch_tiles8<X, 64>(a, stream) : launch_tiles8<X, 128>(a, stream);
        if (plan.mt == 16) return D == 64 ? launch_rows8<X, 64, 1>(a, stream) : launch_rows8<X, 128, 1>(a, stream);
        return D == 64 ? launch_rows8<X, 64, 2>(a, stream) : launch_rows8<X, 128, 2>(a, stream);
    };
    return type == RDA_FP16 ? heads(half_t{}) : heads(bf16_t{});
}

}  // extern "C"
