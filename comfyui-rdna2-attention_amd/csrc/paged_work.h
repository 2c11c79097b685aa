// How attention over a paged cache cuts its work and joins it again: the runs that workgroups take, their partials, and what the kernels of
// 16- and 32-bit caches (paged_attention.hip, whose first comment explains the order of the work) and of quantized ones (paged_int8.hip) share.
#pragma once
#include <type_traits>

#include "paged.h"

#define LOG2E 1.4426950408889634f
#define LEAST -3.402823466e38f  // the lowest finite number
#define MAX_SEQUENCES 8192
#define MAX_KEYS ((1L << 31) - (1L << 16))  // of a sequence: a tile past its end keeps 32-bit key numbers

struct PagedArgs {
    const void* q;
    void* o;
    const void *k, *v;
    const int *table, *starts, *lengths, *prefix;
    const float* slopes;
    char* ws;
    int T, B, H, Hkv, P, N, capacity;  // rows, sequences, heads, KV heads, pages, pages per sequence, N x page size
    Div S, G;                          // page size, query heads per KV head
    Div runs;                          // grid
    long pitch, sqt, sqh, sot, soh, kph, vph;
    u32 kpp, kpr, vpp, vpr;  // strides of pages and of rows: products of them with a 32-bit number are one instruction
    float scale;     // scale log2 e, or scale / cap x 2 log2 e (the exponent of tanh)
    float cap;       // cap log2 e, or 0
    int window, grid, fill;
};

// ------------------------------------------------------------------------------------------------ the order of the work

// A tile: rows r0 .. r1 of a sequence and the keys lo .. hi that any of them sees, in units of UK from lo (a multiple of UK). Its `units` are
// AHEAD more than those of its keys, for what a tile costs before its first key; a run that would end or begin within the first AHEAD ends
// or begins at the tile's start.
struct WorkTile {
    int first, rows;  // the sequence's first row of q; its rows (tokens x heads)
    int r0, r1;       // the tile's rows, r1 included
    int p0;           // position of its token 0 (negative: the length is below the new tokens')
    int keys, prefix; // the sequence's cached keys; those every row sees
    int lo, hi, units;
    int head, skip;   // SKIP: keys left out behind the first `head` units (a multiple of UK)
};

__device__ __forceinline__ int seq_rows(const PagedArgs& p, int b, int& first) {
    first = min(max(p.starts[b], 0), p.T);
    const int end = min(max(p.starts[b + 1], first), p.T);
    return (end - first) * (int)p.G.d;
}
// What a tile costs before its first key, in units: us at 0 / 6 / 8 / 12 units for 24 heads x 4096 causal tokens 281 / 228 / 208 / 200, for a
// chunk of 1001 beside 30 single tokens 95 / 76 / 74 / 74, for 20 ragged chunks over caches 187 / 143 / 135 / 137 (at 10: 143); with changed
// scores, whose units take longer, at 3 / 4 / 6: 2 x 4096 capped in a window 225 / 214 / 213, 5 biased prompts 62 / 62 / 63. Tiles of
// 16 rows at 0 / 1 / 2: 61 single tokens of ragged lengths 144.7 / 140.3 / 142.0, 32 sequences of 5 tokens 130 / 123 / 130. (Times of the code that
// the choice was made on; the 24 heads take 190 now.)
__host__ __device__ constexpr int ahead(int mt, bool mod) { return mt == 128 ? (mod ? 4 : 8) : 1; }
template <int MT, int UK, int AHEAD, bool SKIP = false>
__device__ __forceinline__ WorkTile make_tile(const PagedArgs& p, int b, int j) {
    WorkTile t;
    t.rows = seq_rows(p, b, t.first);
    const int length = max(p.lengths[b], 0), tokens = div_by(t.rows, p.G);
    t.r0 = j * MT;
    t.r1 = min(t.r0 + MT, t.rows) - 1;
    t.p0 = length - tokens;
    t.keys = min(length, p.capacity);
    t.prefix = p.prefix ? min(max(p.prefix[b], 0), t.keys) : 0;
    const int n0 = t.p0 + div_by(t.r0, p.G), n1 = t.p0 + div_by(max(t.r1, 0), p.G);
    t.hi = min(t.keys, max(n1 + 1, t.prefix));
    // With a prefix a tile's keys begin at 0, and without SKIP (16- and 32-bit caches) those between the prefix and the window are walked too, though no row sees them: over 65536 keys
    // with a window of 4096 a single token takes 14 us, with a prefix of 4 keys as well 57, a chunk of 512 tokens 78 and 522.
    t.lo = p.window > 0 && t.prefix == 0 && n0 >= p.window ? (n0 - p.window + 1) / UK * UK : 0;
    t.head = t.skip = 0;
    if constexpr (SKIP) {
        // SKIP (quantized caches) leaves them out: the first `head` units are the prefix's, the others begin where the tile's first row's window does (12.5 and 69 us).
        if (p.window > 0 && t.prefix > 0 && n0 >= p.window) {
            t.head = (t.prefix + UK - 1) / UK;
            // Where the window begins behind the keys (lengths past the table's capacity), up to their end: the units are then the prefix's.
            t.skip = max(min((n0 - p.window + 1) / UK, (t.hi + UK - 1) / UK) - t.head, 0) * UK;
        }
    }
    t.units = AHEAD + max((t.hi - t.lo - t.skip + UK - 1) / UK, 1);  // a tile without keys is one unit: its rows are written too
    return t;
}

// The first unit i whose keys first + i UK and on are all within the window of a row at position n1 (no window: 0). In 64 bits: positions may be up to the
// last of 32 bits, far behind the keys that a short table holds.
template <int UK>
__device__ __forceinline__ int first_unit_in_window(int n1, int window, int first) {
    const long behind = (long)n1 - window + UK - first;
    return window > 0 && behind > 0 ? (int)(behind / UK) : 0;
}

// The same in every lane, which the compiler does not see of values that come from memory: in scalar registers.
__device__ __forceinline__ int uniform(int x) { return __builtin_amdgcn_readfirstlane(x); }
template <class X>
__device__ __forceinline__ const X* uniform(const X* p) {
    const unsigned long long u = (unsigned long long)p;
    return (const X*)((unsigned long long)(u32)uniform((int)(u >> 32)) << 32 | (u32)uniform((int)u));
}
__device__ __forceinline__ WorkTile uniform(WorkTile t) {
    return {uniform(t.first), uniform(t.rows), uniform(t.r0), uniform(t.r1), uniform(t.p0), uniform(t.keys), uniform(t.prefix), uniform(t.lo), uniform(t.hi), uniform(t.units), uniform(t.head), uniform(t.skip)};
}

// Inclusive sums over a wave's lanes, and over the workgroup's NT values (red holds NT / 64 sums).
template <int CTRL, int ROWS>
__device__ __forceinline__ u32 add_from(u32 x) { return x + (u32)__builtin_amdgcn_update_dpp(0, (int)x, CTRL, ROWS, 0xF, false); }
__device__ __forceinline__ u32 scan_wave(u32 x) {
    x = add_from<0x111, 0xF>(x);  // row_shr 1, 2, 4, 8: within 16 lanes
    x = add_from<0x112, 0xF>(x);
    x = add_from<0x114, 0xF>(x);
    x = add_from<0x118, 0xF>(x);
    x = add_from<0x142, 0xA>(x);  // lane 15 of rows 0 and 2 to rows 1 and 3
    return add_from<0x143, 0xC>(x);  // lane 31 to rows 2 and 3
}
template <int NT>
__device__ __forceinline__ u32 scan_block(u32 x, u32* red) {
    const int wave = threadIdx.x >> 6;
    x = scan_wave(x);
    if ((threadIdx.x & 63) == 63) red[wave] = x;
    __syncthreads();
    for (int w = 0; w < wave; w++) x += red[w];
    __syncthreads();
    return x;
}

// Where a workgroup's run begins (KV head, sequence, tile, unit) and how many units it has; 0: none.
struct Run {
    int kvh, b, j, unit, tiles;  // tiles: of sequence b
    int count;
    u32 quota;  // units of every run but the last
};
// The run of workgroup `block` of per_head units a KV head: its KV head and how many units, and the unit within the KV head (returned);
// count 0: none.
__device__ __forceinline__ u32 cut_run(const PagedArgs& p, u32 per_head, int block, Run& run) {
    const unsigned long long total = (unsigned long long)per_head * p.Hkv;
    unsigned long long u0;
    if (total < (1u << 31) - 65536) {
        run.quota = (u32)div_by((int)total + p.grid - 1, p.runs);
        const u32 at = run.quota * (u32)block;  // below total + quota x grid < 2^32
        if (at >= (u32)total) return 0;
        run.kvh = (int)(at / per_head);
        run.count = (int)min(run.quota, (u32)total - at);
        return at - (u32)run.kvh * per_head;
    }
    run.quota = (u32)((total + p.grid - 1) / p.grid);
    u0 = (unsigned long long)run.quota * block;
    if (u0 >= total) return 0;
    run.kvh = (int)(u0 / per_head);
    run.count = (int)min((unsigned long long)run.quota, total - u0);
    return (u32)(u0 - (unsigned long long)run.kvh * per_head);
}
template <int AHEAD>
__device__ __forceinline__ void begin_at_tile(Run& run) {
    if (run.count > 0 && run.unit <= AHEAD) {
        run.count += run.unit;
        run.unit = 0;
    }
}
// smem: B + 1 tile sums; shared: NT + 8 words.
template <int MT, int UK, int AHEAD, int NT, bool SKIP = false>
__device__ __forceinline__ Run find_run(const PagedArgs& p, int* smem, u32* shared, int block) {
    const int t = threadIdx.x;
    u32* red = shared + NT;
    Run run = {};
    // Up to 64 sequences of up to 64 tiles together: every wave by itself, a lane for each. (The search below takes 3 us of a workgroup's time.)
    if (p.B <= 64) {
        const int lane = t & 63;
        int first;
        const u32 tiles = lane < p.B ? (u32)(seq_rows(p, lane, first) + MT - 1) / MT : 0, end = scan_wave(tiles);
        if ((u32)__builtin_amdgcn_readlane((int)end, 63) <= 64) {
            int b = lane;  // the lane's tile's sequence: the first whose tiles end past it
            if (__any(lane < p.B && tiles != 1)) {
                b = 0;
#pragma unroll
                for (int o = 32; o; o >>= 1)
                    if ((int)__shfl(end, b + o - 1) <= lane) b += o;
            }
            const int before = (int)__shfl(end - tiles, min(b, 63)), all = __builtin_amdgcn_readlane((int)end, 63);
            const u32 units = lane < all ? make_tile<MT, UK, AHEAD, SKIP>(p, b, lane - before).units : 0, upto = scan_wave(units);
            const u32 s = cut_run(p, (u32)__builtin_amdgcn_readlane((int)upto, 63), block, run);
            if (run.count == 0) return run;
            const int at = uniform((int)__builtin_ctzll(__ballot(upto > s)));
            run.kvh = uniform(run.kvh);
            run.count = uniform(run.count);
            run.quota = (u32)uniform((int)run.quota);
            run.b = __builtin_amdgcn_readlane(b, at);
            run.j = at - __builtin_amdgcn_readlane(before, at);
            run.tiles = __builtin_amdgcn_readlane((int)tiles, run.b);
            run.unit = uniform((int)(s - (u32)__builtin_amdgcn_readlane((int)(upto - units), at)));
            begin_at_tile<AHEAD>(run);
            return run;
        }
    }
    // Tiles of the sequences before each one.
    const int per = (p.B + NT - 1) / NT, b0 = min(t * per, p.B), b1 = min(b0 + per, p.B);
    u32 tiles = 0;
    for (int b = b0; b < b1; b++) {
        int first;
        tiles += (seq_rows(p, b, first) + MT - 1) / MT;
    }
    u32 before = scan_block<NT>(tiles, red) - tiles;
    for (int b = b0; b < b1; b++) {
        smem[b] = before;
        int first;
        before += (seq_rows(p, b, first) + MT - 1) / MT;
        if (b == p.B - 1) smem[p.B] = before;
    }
    __syncthreads();
    // Units of the tiles before each thread's share of them.
    const int all = smem[p.B], share = (all + NT - 1) / NT, t0 = min(t * share, all), t1 = min(t0 + share, all);
    int b = 0;
    if (t0 < t1) {
        int hi = p.B;  // the sequence of tile t0: the last with smem[b] <= t0
        while (hi - b > 1) {
            const int mid = (b + hi) >> 1;
            if (smem[mid] <= t0) b = mid;
            else hi = mid;
        }
    }
    const int bt = b;
    u32 units = 0;
    for (int i = t0; i < t1; i++) {
        while (smem[b + 1] <= i) b++;
        units += make_tile<MT, UK, AHEAD, SKIP>(p, b, i - smem[b]).units;
    }
    const u32 upto = scan_block<NT>(units, red), from = upto - units;
    if (t == NT - 1) red[4] = upto;
    if (t == 0) shared[3] = 0;
    __syncthreads();
    const u32 s = cut_run(p, red[4], block, run);
    if (run.count == 0) return run;
    if (units && from <= s && s < upto) {  // one thread
        u32 at = from;
        int bb = bt;
        for (int i = t0; i < t1; i++) {
            while (smem[bb + 1] <= i) bb++;
            const u32 n = make_tile<MT, UK, AHEAD, SKIP>(p, bb, i - smem[bb]).units;
            if (s < at + n) {
                shared[0] = bb;
                shared[1] = i - smem[bb];
                shared[2] = s - at;
                shared[3] = smem[bb + 1] - smem[bb];
                break;
            }
            at += n;
        }
    }
    __syncthreads();
    run.kvh = uniform(run.kvh);
    run.b = uniform((int)shared[0]);
    run.j = uniform((int)shared[1]);
    run.unit = uniform((int)shared[2]);
    run.tiles = uniform((int)shared[3]);
    run.count = run.tiles ? uniform(run.count) : 0;  // no tiles: sums past 32 bits (starts that fall)
    run.quota = (u32)uniform((int)run.quota);
    begin_at_tile<AHEAD>(run);
    __syncthreads();
    return run;
}
// The tile after (b, j) of KV head kvh.
template <int MT>
__device__ __forceinline__ void next_tile(const PagedArgs& p, Run& run) {
    if (++run.j < run.tiles) return;
    run.j = 0;
    do {
        if (++run.b == p.B) {
            run.b = 0;
            if (++run.kvh == p.Hkv) {  // only with sums past 32 bits
                run.count = 0;
                return;
            }
        }
        int first;
        run.tiles = uniform((seq_rows(p, run.b, first) + MT - 1) / MT);
    } while (run.tiles == 0);  // ends: the run has units left, so a tile exists
}

// Workspace: a Cut per workgroup, then two partials per workgroup: that of a tile begun before its run (0), and of one begun in it and
// not ended (1). A partial: O [MT][D], m [MT], l [MT].
struct Cut {
    int more;  // workgroups after this one that hold parts of its unended tile; 0: none
    int kvh, first, rows, r0, pad[3];
};
template <int MT, int D>
__device__ __forceinline__ float* partial(const PagedArgs& p, int block, int which) {
    return (float*)(p.ws + (size_t)p.grid * sizeof(Cut)) + ((size_t)block * 2 + which) * MT * (D + 2);
}
// How far below the maximum m stands (see the top). In the rows kernel a tile's maximum may exceed that by 8: a term is at most 2^15. In the tiles
// kernel by 2: a term is at most 2^11, and the sum of a lane's 16 in a full step, which is what the step looks at, 2^15 (MOST).
template <class T>
__host__ __device__ constexpr float lift(int mt) { return std::is_same<T, half_t>::value ? (mt == 128 ? 9.f : 7.f) : 0.f; }
// The offset of a row of a page.
__device__ __forceinline__ unsigned long long row_at(u32 page, u32 page_stride, u32 row, u32 row_stride) {
    return (unsigned long long)page * page_stride + (unsigned long long)row * row_stride;
}
// The workgroup's place in the order of the work: an XCD (block ids go round the eight of them) takes consecutive ones.
__device__ __forceinline__ int work_block(int grid) {
    const int blk = blockIdx.x, xcd = blk % 8, run = grid / 8, rest = grid % 8;
    return xcd * run + min(xcd, rest) + blk / 8;
}

// ------------------------------------------------------------------------------------------------ scores

// log2(e) cap tanh(s / cap) from e = 2 log2(e) scale / cap s: tanh(y) = 1 - 2 / (1 + 2^(2 log2(e) y)). That is off by a few 2^-24 of cap,
// however small the score: below a 16-bit type's own rounding of P for the caps that models use, but all of the score where the cap is
// 10^6 times as large. FINE, for fp32 and for caps from HIGH_CAP on, takes the odd series up to |y| = 1/4 (to y^9: the next term is below 1e-8 of
// the first): off by 2e-6 of the score.
#define HIGH_CAP 2048.f  // log2(e) cap
template <bool FINE>
__device__ __forceinline__ float capped(float e, float cap) {
    const float t = __builtin_fmaf(-2.f, __builtin_amdgcn_rcpf(1.f + __builtin_amdgcn_exp2f(e)), 1.f);
    if constexpr (FINE) {
        const float y = e * 0.34657359027997264f, z = y * y;  // ln(2) / 2
        float s = 62.f / 2835.f;
        s = __builtin_fmaf(s, z, -17.f / 315.f);
        s = __builtin_fmaf(s, z, 2.f / 15.f);
        s = __builtin_fmaf(s, z, -1.f / 3.f);
        s = __builtin_fmaf(s * z, y, y);
        return cap * (fabsf(y) < 0.25f ? s : t);
    }
    return cap * t;
}

// D / 16 consecutive values of a row, divided by the row's sum; a row that saw nothing (its sum 0) is 0.
template <class T, int D>
__device__ __forceinline__ void store_row(T* out, const float (&y)[D / 16], float sum) {
    const float inv = sum == 0.f ? 0.f : 1.f / sum;
    if constexpr (D == 128) {
        f8 x;
#pragma unroll
        for (int e = 0; e < 8; e++) x[e] = y[e] * inv;
        store8(out, x);
    } else {
        typedef T t4 __attribute__((ext_vector_type(4)));
        *(t4*)out = __builtin_convertvector((f4){y[0] * inv, y[1] * inv, y[2] * inv, y[3] * inv}, t4);
    }
}

// ------------------------------------------------------------------------------------------------ tiles of 128 rows

template <int D>
struct TilesLds {
    static constexpr int ROW = 2 * D, TILE = 32 * ROW, V = 3 * TILE;  // K stages, V stages
    // find_run's tile sums before them and the rows turned around after them (32 x 256 bytes a wave) lie in the same place; then find_run's words.
    static constexpr int SHARED = 6 * TILE > 33024 ? 6 * TILE : 33024;
    static_assert(SHARED >= 4 * (MAX_SEQUENCES + 1) && SHARED >= 4 * 32 * 256 && SHARED % 256 == 0);
    static constexpr int BYTES = SHARED + (256 + 16) * 4;
};
typedef __fp16 tr_t __attribute__((__vector_size__(4 * sizeof(__fp16))));
typedef __attribute__((address_space(3))) tr_t lds_tr_t;
typedef __attribute__((address_space(3))) u4v lds_u4v_t;
__device__ __forceinline__ u4v lds_u4(u32 addr) { return *(const lds_u4v_t*)(size_t)addr; }
__device__ __forceinline__ u2v lds_tr(u32 addr) { return __builtin_bit_cast(u2v, __builtin_amdgcn_ds_read_tr16_b64_v4f16((lds_tr_t*)(size_t)addr)); }
__device__ __forceinline__ f2 both_halves(float x) {  // x of the lane's row from lanes 0-31, and from lanes 32-63
    const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return (f2){__uint_as_float(r[0]), __uint_as_float(r[1])};
}
template <class T>
__device__ __forceinline__ f16v product32(const u4v& a, const u4v& b, const f16v& c) {
    if constexpr (std::is_same<T, half_t>::value) return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(h8, a), __builtin_bit_cast(h8, b), c, 0, 0, 0);
    else return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(b8, a), __builtin_bit_cast(b8, b), c, 0, 0, 0);
}
// Two values rounded to T as one word, and the sum of a word's two values added to l.
template <class T>
__device__ __forceinline__ u32 pair_of(float a, float b) {
    if constexpr (std::is_same<T, half_t>::value) return __builtin_bit_cast(u32, __builtin_convertvector((f2){a, b}, h2));
    else return __builtin_bit_cast(u32, __builtin_convertvector((f2){a, b}, b2));
}
template <class T>
__device__ __forceinline__ float add_pair(u32 w, float l) {
    if constexpr (std::is_same<T, half_t>::value) return __builtin_amdgcn_fdot2(__builtin_bit_cast(h2, w), (h2){(_Float16)1.f, (_Float16)1.f}, l, false);
    else return __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(b2, w), (b2){(bf16_t)1.f, (bf16_t)1.f}, l, false);
}

// The lane's number, read again where a rare branch needs it, so that the tile loop holds no registers for it.
__device__ __forceinline__ int lane_again() {
    int x;
    asm volatile("v_mbcnt_lo_u32_b32 %0, -1, 0\n\tv_mbcnt_hi_u32_b32 %0, -1, %0" : "=v"(x));
    return x;
}

// ------------------------------------------------------------------------------------------------ joining

// Adds up the parts of the tiles that the runs cut: workgroups (x, *) those of the tile that run x began and did not end, 16 lanes to a
// row. Of few rows (MT <= 32: single tokens, whose caches are cut into many parts) a wave takes one, each group of 16 lanes every fourth
// part, and the four sums meet; of 128 (cut in two or three) a wave takes four. Also zeroes the rows of no sequence, where the output was
// made for the call. Bound by the partials it reads (66 KB for each cut of a 128-row tile): 18 us behind a chunk of 2048 tokens, 9 behind five
// short prompts; 3.5 to 5.5 us behind single tokens, a launch's and three loads' latency.
template <class T, int D, int MT>
__device__ __forceinline__ void merge_parts(const PagedArgs& p) {
    constexpr bool MANY = MT <= 32;  // parts
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, g = lane >> 4, c = (lane & 15) * (D / 16);
    if (p.fill && blockIdx.y == 0) {
        const int head = min(max(p.starts[0], 0), p.T), tail = min(max(p.starts[p.B], head), p.T);
        for (int i = blockIdx.x; i < head + p.T - tail; i += p.grid) {
            T* row = (T*)p.o + (long)(i < head ? i : i - head + tail) * p.sot;
            for (int x = threadIdx.x; x < p.H * (D / 8); x += 256) store8(row + x / (D / 8) * p.soh + x % (D / 8) * 8, (f8){});
        }
    }
    const Cut cut = ((const Cut*)p.ws)[blockIdx.x];
    const int tr = MANY ? blockIdx.y * 4 + wave : blockIdx.y * 16 + wave * 4 + g, row = cut.r0 + tr;
    if (cut.more == 0 || row >= cut.rows) return;
    const int more = min(cut.more, p.grid - 1 - (int)blockIdx.x);
    auto part_of = [&](int i) __attribute__((always_inline)) { return (const float*)partial<MT, D>(p, blockIdx.x + i, i == 0); };
    float top = -__builtin_inff(), sum = 0.f, y[D / 16];
    float base;
    if constexpr (MANY) {
        for (int i = lane; i <= more; i += 64) top = fmaxf(top, part_of(i)[MT * D + tr]);
        top = rows_max(row_max16(top));
        base = top == -__builtin_inff() ? 0.f : top;
        for (int i = lane; i <= more; i += 64) sum = __builtin_fmaf(part_of(i)[MT * D + MT + tr], __builtin_amdgcn_exp2f(part_of(i)[MT * D + tr] - base), sum);
        sum = rows_sum(row_sum16(sum));
    } else {
#pragma unroll 4
        for (int i = 0; i <= more; i++) top = fmaxf(top, part_of(i)[MT * D + tr]);
        base = top;
    }
#pragma unroll
    for (int e = 0; e < D / 16; e++) y[e] = 0.f;
#pragma unroll 4
    for (int i = MANY ? g : 0; i <= more; i += MANY ? 4 : 1) {
        const float* part = part_of(i);
        const float a = __builtin_amdgcn_exp2f(part[MT * D + tr] - base);
        if constexpr (!MANY) sum = __builtin_fmaf(part[MT * D + MT + tr], a, sum);
#pragma unroll
        for (int e = 0; e < D / 16; e += 4) {
            const f4 z = *(const f4*)(part + tr * D + c + e);
#pragma unroll
            for (int k = 0; k < 4; k++) y[e + k] = __builtin_fmaf(z[k], a, y[e + k]);
        }
    }
    if constexpr (MANY) {
#pragma unroll
        for (int e = 0; e < D / 16; e++) y[e] = rows_sum(y[e]);
        if (g != 0) return;
    }
    const int token = div_by(row, p.G), head = cut.kvh * (int)p.G.d + row - token * (int)p.G.d;
    T* out = (T*)p.o + (long)(cut.first + token) * p.sot + head * p.soh + c;
    store_row<T, D>(out, y, sum);
}
