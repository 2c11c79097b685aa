// Attention of new tokens over a paged key/value cache: sequences of any lengths in one call, one new token each (decode) or many
// (chunks of prompts), in fp16, bf16 or fp32.
//
// Row n of a sequence (its position) with query head h sees keys j <= n (in a window, those with n - j < window; with a prefix, also
// j < prefix). Its scores, in the log2 domain, are x = log2(e) (scale q.k), or log2(e) cap tanh(scale q.k / cap), less log2(e)
// slope_h |n - j|; out = sum_j 2^(x_j - m) v_j / sum_j 2^(x_j - m) in one pass over the keys, m the running maximum. m moves only when
// a tile's maximum exceeds it by more than 8: the terms then stay below 2^8, far inside fp16's range, and O is seldom rescaled. A row
// that sees nothing (or only scores of -inf) is 0.
//
// Work. The query heads of a KV head share its keys: the rows of (sequence, KV head) are its (token, head) pairs in token order, MT
// to a tile, so that single tokens of a group of heads fill a tile with no key read twice. A tile walks the keys that any of its rows
// sees in units of UK keys. All units of a call, ordered by (KV head, sequence, tile, key), are cut into equal runs, one per
// workgroup: a workgroup's run may begin and end inside a tile, and what it finds there goes to the workspace as (O, m, l) partials,
// which a second launch adds up in key order. So long caches of few sequences, ragged batches and causal chunks all balance, with
// nothing but sizes known on the host (lengths are read on the device: a captured launch stays valid as they grow), and with sums in a
// fixed order. KV heads come first in the order and each XCD takes consecutive runs, so that an XCD's L2 holds few heads.
//
// What the pages hold where no row may look (behind a sequence's end, pages the cache does not have) is never used, whatever it
// is: scores are replaced, not added to, and values there are replaced by zeros. Where some rows of a tile see a key that others
// do not, a value that is not finite is added to the rows that see it alone (0 x inf would reach the others).
#include <type_traits>

#include "paged.h"

#define LOG2E 1.4426950408889634f
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
    long pitch, sqt, sqh, sot, soh, kpp, kpr, kph, vpp, vpr, vph;
    float scale;     // scale log2 e, or scale / cap x 2 log2 e (the exponent of tanh)
    float cap;       // cap log2 e, or 0
    int window, grid, fill;
};

// ------------------------------------------------------------------------------------------------ the order of the work

// A tile: rows r0 .. r1 of a sequence and the keys lo .. hi that any of them sees, in units of UK from lo (a multiple of UK).
struct WorkTile {
    int first, rows;  // the sequence's first row of q; its rows (tokens x heads)
    int r0, r1;       // the tile's rows, r1 included
    int p0;           // position of its token 0 (negative: the length is below the new tokens')
    int keys, prefix; // the sequence's cached keys; those every row sees
    int lo, hi, units;
};

__device__ __forceinline__ int seq_rows(const PagedArgs& p, int b, int& first) {
    first = min(max(p.starts[b], 0), p.T);
    const int end = min(max(p.starts[b + 1], first), p.T);
    return (end - first) * (int)p.G.d;
}
template <int MT, int UK>
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
    t.lo = p.window > 0 && t.prefix == 0 && n0 >= p.window ? (n0 - p.window + 1) / UK * UK : 0;
    t.units = max((t.hi - t.lo + UK - 1) / UK, 1);  // a tile without keys is one unit: its rows are written too
    return t;
}

// Inclusive sums over the workgroup's NT values; red holds NT / 64 sums.
template <int NT>
__device__ __forceinline__ u32 scan_block(u32 x, u32* red) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
        const u32 y = __shfl_up(x, o);
        if (lane >= o) x += y;
    }
    if (lane == 63) red[wave] = x;
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
// smem: B + 1 tile sums; shared: NT + 8 words.
template <int MT, int UK, int NT>
__device__ Run find_run(const PagedArgs& p, int* smem, u32* shared, int block) {
    const int t = threadIdx.x;
    u32* red = shared + NT;
    Run run = {};
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
        units += make_tile<MT, UK>(p, b, i - smem[b]).units;
    }
    const u32 upto = scan_block<NT>(units, red), from = upto - units;
    if (t == NT - 1) red[4] = upto;
    if (t == 0) shared[3] = 0;
    __syncthreads();
    const u32 per_head = red[4];
    const unsigned long long total = (unsigned long long)per_head * p.Hkv;
    const u32 quota = (u32)((total + p.grid - 1) / p.grid);
    const unsigned long long u0 = (unsigned long long)quota * block;
    if (u0 >= total) return run;
    const u32 head = (u32)(u0 / per_head), s = (u32)(u0 % per_head);
    if (units && from <= s && s < upto) {  // one thread
        u32 at = from;
        int bb = bt;
        for (int i = t0; i < t1; i++) {
            while (smem[bb + 1] <= i) bb++;
            const u32 n = make_tile<MT, UK>(p, bb, i - smem[bb]).units;
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
    run.kvh = head;
    run.b = __builtin_amdgcn_readfirstlane(shared[0]);
    run.j = __builtin_amdgcn_readfirstlane(shared[1]);
    run.unit = __builtin_amdgcn_readfirstlane(shared[2]);
    run.tiles = __builtin_amdgcn_readfirstlane(shared[3]);
    run.count = run.tiles ? (int)min((unsigned long long)quota, total - u0) : 0;  // no tiles: sums past 32 bits (starts that fall)
    run.quota = quota;
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
        run.tiles = (seq_rows(p, run.b, first) + MT - 1) / MT;
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
// The workgroup's place in the order of the work: an XCD (block ids go round the eight of them) takes consecutive ones.
__device__ __forceinline__ int work_block(int grid) {
    const int blk = blockIdx.x, xcd = blk % 8, run = grid / 8, rest = grid % 8;
    return xcd * run + min(xcd, rest) + blk / 8;
}

// ------------------------------------------------------------------------------------------------ scores

// log2(e) cap tanh(s / cap) from e = 2 log2(e) scale / cap s: tanh(y) = 1 - 2 / (1 + 2^(2 log2(e) y)). Its error of ~1e-7 cap is far below
// a 16-bit type's; fp32 takes the odd series up to |y| = 1/4 (to y^9: the next term is below 1e-8 of the first).
template <bool FP32>
__device__ __forceinline__ float capped(float e, float cap) {
    const float t = __builtin_fmaf(-2.f, __builtin_amdgcn_rcpf(1.f + __builtin_amdgcn_exp2f(e)), 1.f);
    if constexpr (FP32) {
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

// ------------------------------------------------------------------------------------------------ few rows

// Rows kernel: tiles of 16 MB rows, for single tokens and short chunks (and fp32), bound by the keys and values read. Its four waves take
// turns over the keys, KT at a time, and keep everything in registers, K and V loaded straight into the matrix operands:
//
// S^T = K Q^T (16x16 blocks): lane l has row l % 16 of A (a key) and column l % 16 of B (a query row), contraction values of its
// lane group g = l / 16, and of the result column l % 16, rows 4 g .. 4 g + 3. O^T = V^T P^T then has P in the same lanes that
// computed it: with block c's row 4 g + i standing for key KG g + 4 c + i of the tile (KG = 8, two blocks; fp32 4, one block), lane
// group g holds the scores of KG consecutive keys, which are its contraction values in the second product. Row r of A there stands for
// dims VC r + j in product j (VC = D / 16; fp32 4), so that a lane's V operands are VC consecutive dims of KG keys: it loads whole
// rows with its 15 neighbours and pairs two keys' values with a byte permute each. No LDS, no barrier, no lane exchange but the maximum's.
// A page of a multiple of KG keys holds a lane's keys together: one table entry per lane and tile for each of K and V, else one per key.
//
// K of the next tile is loaded as soon as the scores are computed, V as soon as O is: 16 KiB in flight for each of the CU's eight to twelve
// waves, where the memory's latency at full rate needs ~32 KiB per CU.
template <class T>
struct RowsTile {
    static constexpr bool FP32 = sizeof(T) == 4;
    static constexpr int KT = FP32 ? 16 : 32;  // keys of a wave's tile
    static constexpr int KG = KT / 4;          // keys of a lane group
    static constexpr int UK = 4 * KT;          // keys of a unit
};

template <class T, int D, int MB, bool MOD>
__global__ __launch_bounds__(256, MB == 1 && D == 64 ? 3 : 2) void rows_kernel(PagedArgs p) {
    using R = RowsTile<T>;
    constexpr bool FP32 = R::FP32;
    constexpr int KT = R::KT, KG = R::KG, UK = R::UK, MT = 16 * MB;
    constexpr int NB = KG / 4;              // score blocks of 16 keys
    constexpr int EV = 16 / sizeof(T);      // values of a 16-byte vector
    constexpr int KC = D / (4 * EV);        // 16-byte vectors of a lane's part of a K row
    constexpr int VC = FP32 ? 4 : D / 16;   // consecutive dims of a lane's part of a V row
    constexpr int VH = D / (16 * VC);       // such parts
    constexpr int OP = D + 4;               // pitch of a row of O in LDS
    typedef typename std::conditional<FP32, f4, u4v>::type kvec;
    typedef typename std::conditional<FP32, f4, typename std::conditional<VC == 8, u4v, u2v>::type>::type vvec;
    extern __shared__ __attribute__((aligned(16))) char smem[];
    __shared__ u32 shared[256 + 8];
    __shared__ float ml[2][4][16];
    const int t = threadIdx.x, lane = t & 63, g = lane >> 4, r = lane & 15;
    const int wave = __builtin_amdgcn_readfirstlane(t >> 6);
    const int block = work_block(p.grid);
    Run run = find_run<MT, UK, 256>(p, (int*)smem, shared, block);
    Cut cut = {};

    while (run.count > 0) {
        const WorkTile w = make_tile<MT, UK>(p, run.b, run.j);
        const int u0 = run.unit, u1 = min(w.units, u0 + run.count), n = u1 - u0;
        const bool whole = u0 == 0 && u1 == w.units;
        const int* table = p.table + run.b * p.pitch;
        const T* kbase = (const T*)p.k + run.kvh * p.kph;
        const T* vbase = (const T*)p.v + run.kvh * p.vph;

        // Q as the B operand: row r of block m, in the K rows' order of values. pos: the row's position (rows past the tile see nothing).
        kvec qf[MB][KC];
        int pos[MB], pre[MB];
        float slope[MB];
#pragma unroll
        for (int m = 0; m < MB; m++) {
            const int row = w.r0 + 16 * m + r, rc = min(row, w.r1), token = div_by(rc, p.G), head = run.kvh * (int)p.G.d + rc - token * (int)p.G.d;
            const T* src = (const T*)p.q + (long)(w.first + token) * p.sqt + head * p.sqh;
#pragma unroll
            for (int c = 0; c < KC; c++) qf[m][c] = *(const kvec*)(src + (4 * c + g) * EV);
            pos[m] = row <= w.r1 ? w.p0 + token : -1;
            pre[m] = row <= w.r1 ? w.prefix : 0;
            slope[m] = MOD && p.slopes ? p.slopes[head] * LOG2E : 0.f;
        }
        const int n0 = w.p0 + div_by(w.r0, p.G), n1 = w.p0 + div_by(w.r1, p.G);

        f4 o[MB][VH][VC];
        float m_[MB], l_[MB];
#pragma unroll
        for (int m = 0; m < MB; m++) {
#pragma unroll
            for (int h = 0; h < VH; h++)
#pragma unroll
                for (int j = 0; j < VC; j++) o[m][h][j] = (f4){};
            m_[m] = -__builtin_inff();
            l_[m] = 0.f;
        }

        if (w.hi > w.lo) {
            const bool runs = p.S.d % KG == 0;  // a lane group's keys share a page
            // Table entries of tile i: of the lane's K keys and of its V keys.
            auto key_of = [&](int i) __attribute__((always_inline)) { return w.lo + (u0 + i) * UK + wave * KT; };
            int kid[NB], vid[KG];
            auto fetch_ids = [&](int i) __attribute__((always_inline)) {
                const int key0 = key_of(i);
                if (runs) {
                    const int last = (w.hi - 1) / KG * KG;
                    kid[0] = table[div_by(min(key0 + KG * (r >> 2), last), p.S)];
                    vid[0] = table[div_by(min(key0 + KG * g, last), p.S)];
                } else {
#pragma unroll
                    for (int c = 0; c < NB; c++) kid[c] = table[div_by(min(key0 + KG * (r >> 2) + 4 * c + (r & 3), w.hi - 1), p.S)];
#pragma unroll
                    for (int i = 0; i < KG; i++) vid[i] = table[div_by(min(key0 + KG * g + i, w.hi - 1), p.S)];
                }
            };
            // Row of a key, and the first row of its page's entry, with pages that the cache does not have read as page 0.
            auto page_of = [&](int id) __attribute__((always_inline)) { return (u32)id < (u32)p.P ? id : 0; };
            kvec kf[NB][KC];
            vvec vf[KG][VH];
            auto load_k = [&](int i) __attribute__((always_inline)) {
                const int key0 = key_of(i), last = (w.hi - 1) / KG * KG;
#pragma unroll
                for (int c = 0; c < NB; c++) {
                    const int key = runs ? min(key0 + KG * (r >> 2), last) + 4 * c + (r & 3) : min(key0 + KG * (r >> 2) + 4 * c + (r & 3), w.hi - 1);
                    const int row = key - div_by(key, p.S) * (int)p.S.d;
                    const T* src = kbase + page_of(kid[runs ? 0 : c]) * p.kpp + row * p.kpr + g * EV;
#pragma unroll
                    for (int x = 0; x < KC; x++) kf[c][x] = *(const kvec*)(src + 4 * EV * x);
                }
            };
            u32 vbad = 0;  // the lane's V keys on pages the cache does not have
            auto load_v = [&](int i) __attribute__((always_inline)) {
                const int key0 = key_of(i);
                vbad = 0;
                if (runs) {
                    const int key = min(key0 + KG * g, (w.hi - 1) / KG * KG), row = key - div_by(key, p.S) * (int)p.S.d;
                    const T* src = vbase + page_of(vid[0]) * p.vpp + row * p.vpr + r * VC;
                    if ((u32)vid[0] >= (u32)p.P) vbad = ~0u;
#pragma unroll
                    for (int i = 0; i < KG; i++)
#pragma unroll
                        for (int h = 0; h < VH; h++) vf[i][h] = *(const vvec*)(src + i * p.vpr + 16 * VC * h);
                } else {
#pragma unroll
                    for (int i = 0; i < KG; i++) {
                        const int key = min(key0 + KG * g + i, w.hi - 1), row = key - div_by(key, p.S) * (int)p.S.d;
                        const T* src = vbase + page_of(vid[i]) * p.vpp + row * p.vpr + r * VC;
                        if ((u32)vid[i] >= (u32)p.P) vbad |= 1u << i;
#pragma unroll
                        for (int h = 0; h < VH; h++) vf[i][h] = *(const vvec*)(src + 16 * VC * h);
                    }
                }
            };
            fetch_ids(0);
            load_k(0);
            load_v(0);
            u32 bad = vbad;
            if (n > 1) fetch_ids(1);
            for (int i = 0; i < n; i++) {
                const int key0 = key_of(i);
                // Scores.
                float s[MB][KG];
#pragma unroll
                for (int m = 0; m < MB; m++)
#pragma unroll
                    for (int c = 0; c < NB; c++) {
                        f4 acc = {};
#pragma unroll
                        for (int x = 0; x < KC; x++) {
                            if constexpr (FP32) {
#pragma unroll
                                for (int e = 0; e < 4; e++) acc = __builtin_amdgcn_mfma_f32_16x16x4f32(kf[c][x][e], qf[m][x][e], acc, 0, 0, 0);
                            } else if constexpr (std::is_same<T, half_t>::value) {
                                acc = __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(h8, kf[c][x]), __builtin_bit_cast(h8, qf[m][x]), acc, 0, 0, 0);
                            } else {
                                acc = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(b8, kf[c][x]), __builtin_bit_cast(b8, qf[m][x]), acc, 0, 0, 0);
                            }
                        }
#pragma unroll
                        for (int e = 0; e < 4; e++) s[m][4 * c + e] = acc[e] * p.scale;
                    }
                if (i + 1 < n) load_k(i + 1);
                // Whether every row sees every key of the tile.
                const bool all = key0 + KT <= w.hi && !__any(bad != 0) && (key0 + KT <= n0 + 1 || key0 + KT <= w.prefix) &&
                                 (p.window <= 0 || n1 - key0 < p.window || key0 + KT <= w.prefix);
                if constexpr (MOD) {
#pragma unroll
                    for (int m = 0; m < MB; m++)
#pragma unroll
                        for (int e = 0; e < KG; e++) {
                            if (p.cap > 0.f) s[m][e] = capped<FP32>(s[m][e], p.cap);
                            s[m][e] = __builtin_fmaf(-slope[m], fabsf((float)(pos[m] - (key0 + KG * g + e))), s[m][e]);
                        }
                }
                u32 see[MB] = {};
                bool split = false;  // a value that is not finite and that only some rows see
                if (!all) {
#pragma unroll
                    for (int m = 0; m < MB; m++) {
                        see[m] = 0;
#pragma unroll
                        for (int e = 0; e < KG; e++) {
                            const int key = key0 + KG * g + e;
                            const bool there = key < w.hi && !(bad >> e & 1);
                            const bool ok = there && ((key <= pos[m] && (p.window <= 0 || pos[m] - key < p.window)) || key < pre[m]);
                            if (!ok) s[m][e] = -__builtin_inff();
                            see[m] |= ok ? 1u << e : 0;
                        }
                    }
                    // Values at keys that the sequence does not have become zeros; those of the others are looked at.
                    bool odd = false;
#pragma unroll
                    for (int e = 0; e < KG; e++) {
                        const bool there = key0 + KG * g + e < w.hi && !(bad >> e & 1);
#pragma unroll
                        for (int h = 0; h < VH; h++) {
                            if (!there) vf[e][h] = (vvec){};
#pragma unroll
                            for (int x = 0; x < (int)(sizeof(vvec) / 4); x++) {
                                const u32 word = FP32 ? __float_as_uint(vf[e][h][x]) : (u32)vf[e][h][x];
                                if constexpr (FP32) odd |= (word & 0x7f800000u) == 0x7f800000u;
                                else {
                                    constexpr u32 E = std::is_same<T, half_t>::value ? 0x7c00u : 0x7f80u;
                                    odd |= (word & E) == E || (word >> 16 & E) == E;
                                }
                            }
                        }
                    }
                    split = __any(odd);
                }
                // Softmax.
                u4v pf[MB];
                float pw[MB][KG];
#pragma unroll
                for (int m = 0; m < MB; m++) {
                    float mx = s[m][0];
#pragma unroll
                    for (int e = 1; e < KG; e++) mx = fmaxf(mx, s[m][e]);
                    mx = rows_max(mx);
                    const bool move = mx > m_[m] + 8.f || (m_[m] == -__builtin_inff() && mx > m_[m]);
                    if (__any(move)) {
                        const float a = move ? __builtin_amdgcn_exp2f(m_[m] - mx) : 1.f;
                        m_[m] = move ? mx : m_[m];
                        l_[m] *= a;
#pragma unroll
                        for (int h = 0; h < VH; h++)
#pragma unroll
                            for (int j = 0; j < VC; j++) o[m][h][j] *= a;
                    }
                    const float base = m_[m] == -__builtin_inff() ? 0.f : m_[m];
#pragma unroll
                    for (int e = 0; e < KG; e++) pw[m][e] = __builtin_amdgcn_exp2f(s[m][e] - base);
                    if constexpr (FP32) {
#pragma unroll
                        for (int e = 0; e < KG; e++) l_[m] += pw[m][e];
                    } else {
                        // P is rounded to the cache's type for the product, and l sums those values: the weights that are used add up to 1.
                        if constexpr (std::is_same<T, half_t>::value) {
                            h8 x;
#pragma unroll
                            for (int e = 0; e < 8; e++) x[e] = to_half(pw[m][e]), l_[m] += (float)x[e];
                            pf[m] = __builtin_bit_cast(u4v, x);
                        } else {
                            b8 x;
#pragma unroll
                            for (int e = 0; e < 8; e++) x[e] = (bf16_t)pw[m][e];
                            pf[m] = __builtin_bit_cast(u4v, x);
#pragma unroll
                            for (int e = 0; e < 4; e++) l_[m] += __uint_as_float(pf[m][e] << 16) + __uint_as_float(pf[m][e] & 0xffff0000u);
                        }
                    }
                }
                // O^T += V^T P^T.
                auto product = [&](const u4v& a, const u4v& b, const f4& acc) __attribute__((always_inline)) {
                    if constexpr (std::is_same<T, half_t>::value) return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(h8, a), __builtin_bit_cast(h8, b), acc, 0, 0, 0);
                    else return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(b8, a), __builtin_bit_cast(b8, b), acc, 0, 0, 0);
                };
#pragma unroll
                for (int h = 0; h < VH; h++)
#pragma unroll
                    for (int j = 0; j < VC; j++) {
                        if constexpr (FP32) {
                            if (__builtin_expect(!split, 1)) {
#pragma unroll
                                for (int m = 0; m < MB; m++)
#pragma unroll
                                    for (int e = 0; e < 4; e++) o[m][h][j] = __builtin_amdgcn_mfma_f32_16x16x4f32(vf[e][h][j], pw[m][e], o[m][h][j], 0, 0, 0);
                            } else {
                                for (int kk = 0; kk < KT; kk++) {  // one key at a time, into the rows that see it
                                    float a = 0.f;
#pragma unroll
                                    for (int e = 0; e < 4; e++) a = kk == 4 * g + e ? vf[e][h][j] : a;
#pragma unroll
                                    for (int m = 0; m < MB; m++) {
                                        float w1 = 0.f;
#pragma unroll
                                        for (int e = 0; e < 4; e++) w1 = (kk & 3) == e ? pw[m][e] : w1;
                                        const f4 one = __builtin_amdgcn_mfma_f32_16x16x4f32(a, w1, (f4){}, 0, 0, 0);
                                        if (__shfl(see[m] >> (kk & 3) & 1, (kk >> 2) * 16 + r)) o[m][h][j] += one;
                                    }
                                }
                            }
                        } else {
                            u4v a;
#pragma unroll
                            for (int e = 0; e < 4; e++)
                                a[e] = __builtin_amdgcn_perm((u32)vf[2 * e + 1][h][j >> 1], (u32)vf[2 * e][h][j >> 1], j & 1 ? 0x07060302u : 0x05040100u);
                            if (__builtin_expect(!split, 1)) {
#pragma unroll
                                for (int m = 0; m < MB; m++) o[m][h][j] = product(a, pf[m], o[m][h][j]);
                            } else {
                                for (int kk = 0; kk < KT; kk++) {
                                    u4v one_key;
#pragma unroll
                                    for (int e = 0; e < 4; e++) one_key[e] = kk >> 1 == 4 * g + e ? a[e] & (kk & 1 ? 0xffff0000u : 0xffffu) : 0;
#pragma unroll
                                    for (int m = 0; m < MB; m++) {
                                        const f4 one = product(one_key, pf[m], (f4){});
                                        if (__shfl(see[m] >> (kk & 7) & 1, (kk >> 3) * 16 + r)) o[m][h][j] += one;
                                    }
                                }
                            }
                        }
                    }
                if (i + 1 < n) {
                    load_v(i + 1);
                    bad = vbad;
                    if (i + 2 < n) fetch_ids(i + 2);
                }
            }
        }

        // The four waves' results meet in LDS, 16 rows at a time: thread (row t / 16, dims from t % 16 on) adds them.
#pragma unroll
        for (int m = 0; m < MB; m++) {
            const float l = rows_sum(l_[m]);
            __syncthreads();
            if (g == 0) {
                ml[0][wave][r] = m_[m];
                ml[1][wave][r] = l;
            }
            float* dst = (float*)smem + (wave * 16 + r) * OP;
#pragma unroll
            for (int h = 0; h < VH; h++)
#pragma unroll
                for (int i = 0; i < 4; i++)  // dims 16 VC h + VC (4 g + i) + j
#pragma unroll
                    for (int j = 0; j < VC; j += 4)
                        *(f4*)(dst + 16 * VC * h + VC * (4 * g + i) + j) = (f4){o[m][h][j][i], o[m][h][j + 1][i], o[m][h][j + 2][i], o[m][h][j + 3][i]};
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
                    const float inv = sum == 0.f ? 0.f : 1.f / sum;
#pragma unroll
                    for (int e = 0; e < D / 16; e++) out[e] = sum == 0.f ? (T)0.f : (T)(y[e] * inv);
                }
            } else {
                float* part = partial<MT, D>(p, block, u0 == 0);
#pragma unroll
                for (int e = 0; e < D / 16; e += 4) *(f4*)(part + tr * D + c + e) = (f4){y[e], y[e + 1], y[e + 2], y[e + 3]};
                if (c == 0) {
                    part[MT * D + tr] = top;
                    part[MT * D + MT + tr] = sum;
                }
            }
        }
        __syncthreads();
        if (u0 == 0 && u1 < w.units) {
            cut.more = (int)((w.units - u1 + run.quota - 1) / run.quota);
            cut.kvh = run.kvh;
            cut.first = w.first;
            cut.rows = w.rows;
            cut.r0 = w.r0;
        }
        run.count -= n;
        run.unit = 0;
        if (run.count > 0) next_tile<MT>(p, run);
    }
    if (t == 0) ((Cut*)p.ws)[block] = cut;
}

// Adds up the parts of the tiles that the runs cut: workgroup (x, y) takes rows 4 y .. 4 y + 3 of the tile that run x began and did not
// end, a wave per row; lanes 16 i .. 16 i + 15 take every fourth part from the i-th on, then the four sums meet. Also zeroes the rows
// of no sequence, where the output was made for the call.
template <class T, int D, int MT>
__global__ __launch_bounds__(256) void merge_kernel(PagedArgs p) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, g = lane >> 4, c = (lane & 15) * (D / 16);
    if (p.fill && blockIdx.y == 0) {
        const int head = min(max(p.starts[0], 0), p.T), tail = min(max(p.starts[p.B], head), p.T);
        for (int i = blockIdx.x; i < head + p.T - tail; i += p.grid) {
            T* row = (T*)p.o + (long)(i < head ? i : i - head + tail) * p.sot;
            for (int x = threadIdx.x; x < p.H * (D / 8); x += 256) store8(row + x / (D / 8) * p.soh + x % (D / 8) * 8, (f8){});
        }
    }
    const Cut cut = ((const Cut*)p.ws)[blockIdx.x];
    const int tr = blockIdx.y * 4 + wave, row = cut.r0 + tr;
    if (cut.more == 0 || row >= cut.rows) return;
    float top = -__builtin_inff(), sum = 0.f, y[D / 16];
#pragma unroll
    for (int e = 0; e < D / 16; e++) y[e] = 0.f;
    const int more = min(cut.more, p.grid - 1 - (int)blockIdx.x);
    for (int i = g; i <= more; i += 4) {
        const float* part = partial<MT, D>(p, blockIdx.x + i, i == 0);
        const float m = part[MT * D + tr], l = part[MT * D + MT + tr], now = fmaxf(top, m);
        const float a = top == -__builtin_inff() ? 0.f : __builtin_amdgcn_exp2f(top - now), b = m == -__builtin_inff() ? 0.f : __builtin_amdgcn_exp2f(m - now);
        top = now;
        sum = __builtin_fmaf(sum, a, l * b);
#pragma unroll
        for (int e = 0; e < D / 16; e += 4) {
            const f4 z = *(const f4*)(part + tr * D + c + e);
#pragma unroll
            for (int k = 0; k < 4; k++) y[e + k] = __builtin_fmaf(y[e + k], a, z[k] * b);
        }
    }
    const float all = rows_max(top), a = top == -__builtin_inff() ? 0.f : __builtin_amdgcn_exp2f(top - all);
    sum = rows_sum(sum * a);
#pragma unroll
    for (int e = 0; e < D / 16; e++) y[e] = rows_sum(y[e] * a);
    if (g == 0) {
        const int token = div_by(row, p.G), head = cut.kvh * (int)p.G.d + row - token * (int)p.G.d;
        T* out = (T*)p.o + (long)(cut.first + token) * p.sot + head * p.soh + c;
        const float inv = sum == 0.f ? 0.f : 1.f / sum;
#pragma unroll
        for (int e = 0; e < D / 16; e++) out[e] = sum == 0.f ? (T)0.f : (T)(y[e] * inv);
    }
}

// ------------------------------------------------------------------------------------------------ launches

struct Plan {
    int mt, grid;
    size_t workspace;
};
static int make_plan(long T, long B, long H, long Hkv, long D, int type, Plan* plan) {
    if (T <= 0 || B <= 0 || B > MAX_SEQUENCES || Hkv <= 0 || H <= 0 || H % Hkv || (D != 64 && D != 128) || type < RDA_FP16 || type > RDA_FP32) return RDA_ERR_INVALID;
    if (T * (H / Hkv) >= 1L << 31) return RDA_ERR_INVALID;
    // Rows of a sequence and KV head, on average.
    const long rows = T * (H / Hkv) / B;
    plan->mt = rows <= 16 ? 16 : 32;
    plan->grid = plan->mt == 16 ? 768 : 512;
    if ((T * (H / Hkv) / plan->mt + 1) * B >= 1L << 31) return RDA_ERR_INVALID;
    plan->workspace = (size_t)plan->grid * sizeof(Cut) + (size_t)plan->grid * 2 * plan->mt * (D + 2) * 4;
    return 0;
}

template <class T, int D, int MB>
static int launch_rows(const PagedArgs& a, void* stream) {
    constexpr int OP = D + 4;
    const size_t o = 4 * 16 * OP * 4, sums = (size_t)(a.B + 1) * 4, lds = o > sums ? o : sums;
    const bool mod = a.cap > 0.f || a.slopes;
    if (mod) hipLaunchKernelGGL((rows_kernel<T, D, MB, true>), dim3(a.grid), dim3(256), lds, (hipStream_t)stream, a);
    else hipLaunchKernelGGL((rows_kernel<T, D, MB, false>), dim3(a.grid), dim3(256), lds, (hipStream_t)stream, a);
    if (const hipError_t e = hipGetLastError()) return (int)e;
    hipLaunchKernelGGL((merge_kernel<T, D, 16 * MB>), dim3(a.grid, 4 * MB), dim3(256), 0, (hipStream_t)stream, a);
    return (int)hipGetLastError();
}
template <class T, int D>
static int launch_paged(const PagedArgs& a, const Plan& plan, void* stream) {
    return plan.mt == 16 ? launch_rows<T, D, 1>(a, stream) : launch_rows<T, D, 2>(a, stream);
}

static bool vector_rows(const void* p, const long* strides, int n, int type) {
    const long m = type == RDA_FP32 ? 4 : 8;
    for (int i = 0; i < n; i++)
        if (strides[i] % m) return false;
    return ((uintptr_t)p & 15) == 0;
}

extern "C" {

size_t rda_paged_attn_workspace(long T, long B, long H, long Hkv, long D, int type) {
    Plan plan;
    return make_plan(T, B, H, Hkv, D, type, &plan) ? 0 : plan.workspace;
}

int rda_paged_attn(const void* q, void* out, const void* k_pages, const void* v_pages, const int* table, const int* starts, const int* lengths,
                   const int* prefix, const float* slopes, void* workspace, float scale, float softcap, int window, int fill, int type, const long* dims,
                   void* stream) {
    const long T = dims[0], H = dims[1], Hkv = dims[2], D = dims[3], B = dims[4], N = dims[5], P = dims[7], S = dims[8];
    Plan plan;
    if (const int e = make_plan(T, B, H, Hkv, D, type, &plan)) return e;
    if (N <= 0 || P <= 0 || P >= 1L << 31 || S <= 0 || N > MAX_KEYS / S || window < 0 || !(softcap >= 0.f) || ((uintptr_t)workspace & 15)) return RDA_ERR_INVALID;
    if (!vector_rows(q, dims + 9, 2, type) || !vector_rows(out, dims + 11, 2, type) || !vector_rows(k_pages, dims + 13, 3, type) ||
        !vector_rows(v_pages, dims + 16, 3, type))
        return RDA_ERR_INVALID;
    // Units of a KV head in 32 bits, whatever the lengths.
    if ((T * (H / Hkv) / plan.mt + B) * (N * S / 64 + 1) >= 1L << 32) return RDA_ERR_INVALID;
    PagedArgs a;
    a.q = q; a.o = out; a.k = k_pages; a.v = v_pages;
    a.table = table; a.starts = starts; a.lengths = lengths; a.prefix = prefix;
    a.slopes = slopes;
    a.ws = (char*)workspace;
    a.T = (int)T; a.B = (int)B; a.H = (int)H; a.Hkv = (int)Hkv; a.P = (int)P; a.N = (int)N; a.capacity = (int)(N * S);
    a.S = make_div((int)S); a.G = make_div((int)(H / Hkv));
    a.pitch = dims[6];
    a.sqt = dims[9]; a.sqh = dims[10]; a.sot = dims[11]; a.soh = dims[12];
    a.kpp = dims[13]; a.kpr = dims[14]; a.kph = dims[15]; a.vpp = dims[16]; a.vpr = dims[17]; a.vph = dims[18];
    a.scale = softcap > 0.f ? scale / softcap * 2.f * LOG2E : scale * LOG2E;
    a.cap = softcap * LOG2E;
    a.window = window;
    a.grid = plan.grid;
    a.fill = fill;
    const auto heads = [&](auto x) {
        using X = decltype(x);
        return D == 64 ? launch_paged<X, 64>(a, plan, stream) : launch_paged<X, 128>(a, plan, stream);
    };
    return type == RDA_FP16 ? heads(half_t{}) : type == RDA_BF16 ? heads(bf16_t{}) : heads(float{});
}

}  // extern "C"
