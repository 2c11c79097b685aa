// Attention of new tokens over a paged key/value cache: sequences of any lengths in one call, one new token each (decode) or many
// (chunks of prompts), in fp16, bf16 or fp32.
//
// Row n of a sequence (its position) with query head h sees keys j <= n (in a window, those with n - j < window; with a prefix, also
// j < prefix). Its scores, in the log2 domain, are x = log2(e) (scale q.k), or log2(e) cap tanh(scale q.k / cap), less log2(e)
// slope_h |n - j|; out = sum_j 2^(x_j - m) v_j / sum_j 2^(x_j - m) in one pass over the keys, m the running maximum. m moves only when
// a tile's maximum exceeds it by more than 8 (2 in tiles of 128 rows), so that O is seldom rescaled. For an fp16 cache m stands below the
// maximum by lift() and the terms are that much larger, near the top of fp16's range: one of 2^-21 of the largest still has all of
// fp16's bits, where many keys of little weight stand beside one of much. A row that sees nothing (or only scores of -inf) is 0.
// In 16-bit types the terms are rounded to the type, which the second product's matrix instructions take, and the sum is of the rounded terms, so that
// the weights in use add up to 1. Beside the output's own rounding that costs little: rms errors are 1.1 times (single tokens, and fp16) to
// 1.4 times (a bf16 chunk) those of 32-bit terms. Scores, m, l and O are held in 32 bits.
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
#include "paged_work.h"

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
// waves, where the memory's latency at full rate needs ~32 KiB per CU. 64 single tokens over 8192 bf16 keys (8 KV heads of 128): 370 to 386 us
// for 2.1 GB, 5.6 to 5.8 TB/s, where a sum of 1 GiB reads at 6.0. 61 over 1 to 16384 keys: 132 us for 657 MB, 5.0 TB/s: a run there is about two
// tiles, each of which starts and ends with little in flight (~3 us). One fp32 token over 2048 keys: 8 to 9 us of latencies.
template <class T>
struct RowsTile {
    static constexpr bool FP32 = sizeof(T) == 4;
    static constexpr int KT = FP32 ? 16 : 32;  // keys of a wave's tile
    static constexpr int KG = KT / 4;          // keys of a lane group
    static constexpr int UK = 4 * KT;          // keys of a unit
};

template <class T, int D, int MB, bool MOD, bool RUNS>
__global__ __launch_bounds__(256, MB == 1 && D == 64 ? 3 : 2) void rows_kernel(PagedArgs p) {
    using R = RowsTile<T>;
    constexpr bool FP32 = R::FP32;
    constexpr int KT = R::KT, KG = R::KG, UK = R::UK, MT = 16 * MB, AHEAD = ahead(MT, MOD);
    constexpr float LIFT = lift<T>(MT);
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
    Run run = find_run<MT, UK, AHEAD, 256>(p, (int*)smem, shared, block);
    Cut cut = {};

    while (run.count > 0) {
        const WorkTile w = uniform(make_tile<MT, UK, AHEAD>(p, run.b, run.j));
        if (run.unit + run.count <= AHEAD) break;  // the next run's
        const bool begins = run.unit == 0, last_part = run.unit + run.count >= w.units, whole = begins && last_part;
        const int u0 = begins ? 0 : run.unit - AHEAD, u1 = min(w.units, run.unit + run.count) - AHEAD, n = u1 - u0;
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
        const int n0 = uniform(w.p0 + div_by(w.r0, p.G)), n1 = uniform(w.p0 + div_by(w.r1, p.G));

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
            // Table entries of tile i: of the lane's K keys and of its V keys.
            auto key_of = [&](int i) __attribute__((always_inline)) { return w.lo + (u0 + i) * UK + wave * KT; };
            int kid[RUNS ? 1 : NB], vid[RUNS ? 1 : KG];
            auto fetch_ids = [&](int i) __attribute__((always_inline)) {
                const int key0 = key_of(i);
                if constexpr (RUNS) {
                    const int last = (w.hi - 1) / KG * KG;
                    kid[0] = table[div_by(min(key0 + KG * (r >> 2), last), p.S)];
                    vid[0] = table[div_by(min(key0 + KG * g, last), p.S)];
                } else {
#pragma unroll
                    for (int c = 0; c < NB; c++) kid[c] = table[div_by(min(key0 + KG * (r >> 2) + 4 * c + (r & 3), w.hi - 1), p.S)];
#pragma unroll
                    for (int e = 0; e < KG; e++) vid[e] = table[div_by(min(key0 + KG * g + e, w.hi - 1), p.S)];
                }
            };
            // The address of a key's row; pages that the cache does not have are read as page 0.
            auto row_of = [&](const T* base, int id, int key, u32 page_stride, u32 row_stride) __attribute__((always_inline)) {
                const u32 page = (u32)id < (u32)p.P ? (u32)id : 0, row = (u32)(key - div_by(key, p.S) * (int)p.S.d);
                return base + row_at(page, page_stride, row, row_stride);
            };
            kvec kf[NB][KC];
            vvec vf[KG][VH];
            auto load_k = [&](int i) __attribute__((always_inline)) {
                const int key0 = key_of(i);
                if constexpr (RUNS) {
                    const T* src = row_of(kbase, kid[0], min(key0 + KG * (r >> 2), (w.hi - 1) / KG * KG) + (r & 3), p.kpp, p.kpr) + g * EV;
#pragma unroll
                    for (int c = 0; c < NB; c++)
#pragma unroll
                        for (int x = 0; x < KC; x++) kf[c][x] = *(const kvec*)(src + (unsigned long long)(4 * c) * p.kpr + 4 * EV * x);
                } else {
#pragma unroll
                    for (int c = 0; c < NB; c++) {
                        const T* src = row_of(kbase, kid[c], min(key0 + KG * (r >> 2) + 4 * c + (r & 3), w.hi - 1), p.kpp, p.kpr) + g * EV;
#pragma unroll
                        for (int x = 0; x < KC; x++) kf[c][x] = *(const kvec*)(src + 4 * EV * x);
                    }
                }
            };
            u32 vbad = 0;  // the lane's V keys on pages the cache does not have
            auto load_v = [&](int i) __attribute__((always_inline)) {
                const int key0 = key_of(i);
                if constexpr (RUNS) {
                    const T* src = row_of(vbase, vid[0], min(key0 + KG * g, (w.hi - 1) / KG * KG), p.vpp, p.vpr) + r * VC;
                    vbad = (u32)vid[0] < (u32)p.P ? 0 : ~0u;
#pragma unroll
                    for (int e = 0; e < KG; e++)
#pragma unroll
                        for (int h = 0; h < VH; h++) vf[e][h] = *(const vvec*)(src + (unsigned long long)e * p.vpr + 16 * VC * h);
                } else {
                    vbad = 0;
#pragma unroll
                    for (int e = 0; e < KG; e++) {
                        const T* src = row_of(vbase, vid[e], min(key0 + KG * g + e, w.hi - 1), p.vpp, p.vpr) + r * VC;
                        vbad |= (u32)vid[e] < (u32)p.P ? 0 : 1u << e;
#pragma unroll
                        for (int h = 0; h < VH; h++) vf[e][h] = *(const vvec*)(src + 16 * VC * h);
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
                    const auto cap_all = [&](auto fine) __attribute__((always_inline)) {
#pragma unroll
                        for (int m = 0; m < MB; m++)
#pragma unroll
                            for (int e = 0; e < KG; e++) s[m][e] = capped<decltype(fine)::value>(s[m][e], p.cap);
                    };
                    if (FP32 ? p.cap > 0.f : p.cap >= HIGH_CAP) cap_all(std::true_type{});
                    else if (p.cap > 0.f) cap_all(std::false_type{});
#pragma unroll
                    for (int m = 0; m < MB; m++)
#pragma unroll
                        for (int e = 0; e < KG; e++) s[m][e] = __builtin_fmaf(-slope[m], fabsf((float)(pos[m] - (key0 + KG * g + e))), s[m][e]);
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
                    // Values at keys that no row sees become zeros. Where all rows are of one token that is all; else the others are looked at.
                    u32 seen = 0;
#pragma unroll
                    for (int m = 0; m < MB; m++) seen |= see[m];
#pragma unroll
                    for (int o = 1; o < 16; o <<= 1) seen |= __shfl_xor(seen, o);
#pragma unroll
                    for (int e = 0; e < KG; e++)
#pragma unroll
                        for (int h = 0; h < VH; h++)
                            if (!(seen >> e & 1)) vf[e][h] = (vvec){};
                    if (n0 != n1) {
                        bool odd = false;
#pragma unroll
                        for (int e = 0; e < KG; e++)
#pragma unroll
                            for (int h = 0; h < VH; h++)
#pragma unroll
                                for (int x = 0; x < (int)(sizeof(vvec) / 4); x++) {
                                    const auto element = vf[e][h][x];  // (the bit cast of a vector's element itself reads element 0)
                                    const u32 word = __builtin_bit_cast(u32, element);
                                    constexpr u32 E = FP32 ? 0x7f800000u : std::is_same<T, half_t>::value ? 0x7c00u : 0x7f80u;
                                    odd |= (word & E) == E || (!FP32 && (word >> 16 & E) == E);
                                }
                        split = __any(odd);
                    }
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
                    const bool move = mx > m_[m] + (8.f + LIFT) || (m_[m] == -__builtin_inff() && mx > m_[m]);
                    mx -= LIFT;
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

// ------------------------------------------------------------------------------------------------ many rows

// Tiles kernel (fp16, bf16): tiles of 128 rows, 32 to each of four waves, which share 32-key tiles of K and V in LDS. Bound by the
// matrix products and the exponentials beside them, as the fused attention of fixed shapes (attention.hip), whose tile layouts and
// step order it has: S^T = K Q^T and O^T = V^T P^T in 32x32 blocks, a lane's registers all of its own row (lane % 32; the lane
// 32 on has the row's other keys); three stages filled by 16-byte global->LDS copies two tiles ahead; step i computes tile i + 1's scores
// beside tile i's second half of exponentials, then tile i's product with V beside tile i + 1's first half. What differs:
//
// * A copy's rows come from pages. A wave's copy has 4 rows (D = 64: 8) of a tile, in one page where the page size is a multiple of 8:
//   its base is then scalar, else each lane has its own. Table entries are fetched one step before the copies they are for, and have
//   arrived by the barrier that ends it.
// * Tiles at the ends of what the wave's rows see are masked, by a branch that the other tiles skip. Scores are replaced by -inf, and m
//   starts at the lowest finite number, so that a row without keys so far has P = 0.
// * Keys past the sequence's end are copies of its last row, and those on pages that the cache does not have rows of page 0; masked
//   tiles whose values are not all finite add them key by key to the rows that see them.
//
// A chunk of 2048 tokens, 32 heads over 8 KV heads of 128 bf16, over 14336 cached keys: 538 to 554 us for 515 GFLOP, 0.94 PFLOP/s, 69 to 80% of what a
// library product of 8192^3 reaches (1.18 to 1.37 by the box). The matrix instructions run in 47% of the cycles (at 1.6 to 1.9 GHz, the chip's power limit) and five other vector
// instructions stand beside each; the two do not overlap within a wave's SIMD, and add up to nearly all of them. LDS reads meet no bank conflict.
// Capped scores take three transcendentals each where plain ones take one: 2 x 4096 tokens of 16 heads of 128 in a window of 2048, 103 GFLOP, 190 us:
// at two workgroups a CU vector work and products fill ~80% of the cycles (217 us with the whole capped score made before the softmax's product).
// With D = 64 a score's exponential stands beside half the products. Tiles that are masked cost ~2.4 full ones, a tile's start ~7 us of latency.
template <class T, int D, bool MOD, bool RUNS>
__global__ __launch_bounds__(256, D == 128 && MOD ? 2 : 3) void tiles_kernel(PagedArgs p) {
    constexpr int MT = 128, UK = 32, AHEAD = ahead(MT, MOD), ROW = 2 * D, KS = D / 16, DT = D / 32;  // KS: products of a score block; DT: of a 16-key step with V
    constexpr int CP = D / 64, CR = 1024 / ROW;  // a wave's copies of K per tile; rows of a copy
    constexpr float LIFT = lift<T>(MT), MOST = 64.f * (std::is_same<T, half_t>::value ? 512.f : 1.f);  // of a full step's sum of P in a lane: 64 2^LIFT
    using L = TilesLds<D>;
    extern __shared__ __attribute__((aligned(256))) char smem[];
    const int lane = threadIdx.x & 63, g = lane >> 5, lq = lane & 31;
    const int wave = uniform((int)(threadIdx.x >> 6));
    const int block = work_block(p.grid);
    Run run = find_run<MT, UK, AHEAD, 256>(p, (int*)smem, (u32*)(smem + L::SHARED), block);
    int* flags = (int*)(smem + L::SHARED) + 256 + 8;  // a wave's: whether the cache lacks a page that it looked up
    Cut cut = {};
    const u32 smem_u = lds_addr(smem);

    while (run.count > 0) {
        const WorkTile w = uniform(make_tile<MT, UK, AHEAD>(p, run.b, run.j));
        if (run.unit + run.count <= AHEAD) break;  // the next run's
        const bool begins = run.unit == 0, last_part = run.unit + run.count >= w.units, whole = begins && last_part;
        const int u0 = begins ? 0 : run.unit - AHEAD, u1 = min(w.units, run.unit + run.count) - AHEAD, n = w.hi > w.lo ? u1 - u0 : 0;
        const int* table = p.table + run.b * p.pitch;
        const T* kbase = uniform((const T*)p.k + run.kvh * p.kph);
        const T* vbase = uniform((const T*)p.v + run.kvh * p.vph);
        const int key_first = w.lo + u0 * UK;
        auto key_of = [&](int i) __attribute__((always_inline)) { return key_first + i * UK; };
        const int wr0 = w.r0 + 32 * wave;  // the wave's first row
        const bool active = wr0 <= w.r1;
        const int n0 = uniform(w.p0 + div_by(min(wr0, w.r1), p.G)), n1 = uniform(w.p0 + div_by(min(wr0 + 31, w.r1), p.G));

        // Copies. Copy c of a tile: rows CR (4 c + wave) .. + CR - 1, the lane's row at + lane / (D / 8); the 16-byte chunks of a row are
        // permuted in LDS so that reads hit distinct banks: K chunk x of row r at x ^ (r & 15) (D = 64: x ^ (r / 2 & 7)), V chunk at
        // x ^ 4 (r & 3) (D = 64: x ^ 4 (r / 2 & 1)). Copies 1 differ from copies 0 by rows of a multiple of 16: by the base alone.
        auto k_chunk = [](int ln, int r) __attribute__((always_inline)) { return (ln % (D / 8)) ^ (D == 128 ? r & 15 : r >> 1 & 7); };
        auto v_chunk = [](int ln, int r) __attribute__((always_inline)) { return (ln % (D / 8)) ^ (D == 128 ? (r & 3) << 2 : (r >> 1 & 1) << 2); };
        const int my_row = CR * wave + lane / (D / 8);
        u32 k_off = (u32)(lane / (D / 8) * (int)p.kpr * 2 + k_chunk(lane, my_row) * 16), v_off = (u32)(lane / (D / 8) * (int)p.vpr * 2 + v_chunk(lane, my_row) * 16);
        int id[CP];  // table entries of the tile to be copied next: of the lane's rows
        auto fetch = [&](int i) __attribute__((always_inline)) {
            const int ln = lane_again();
#pragma unroll
            for (int c = 0; c < CP; c++) id[c] = table[div_by(min(key_of(i) + CR * (4 * c + wave) + ln / (D / 8), w.hi - 1), p.S)];
        };
        auto issue = [&](int i, u32 st) __attribute__((always_inline)) {
            const int ln = lane_again();
#pragma unroll
            for (int c = 0; c < CP; c++) {
                const int r = CR * (4 * c + wave), lr = r + ln / (D / 8), key = min(key_of(i) + lr, w.hi - 1), kr = key - div_by(key, p.S) * (int)p.S.d;
                const u32 at = (u32)id[c] < (u32)p.P ? id[c] : 0;
                dma16_at(kbase + (row_at(at, p.kpp, kr, p.kpr) + k_chunk(ln, lr) * 8), smem + st + r * ROW);
                dma16_at(vbase + (row_at(at, p.vpp, kr, p.vpr) + v_chunk(ln, lr) * 8), smem + L::V + st + r * ROW);
            }
        };
        // The same for a tile without an end and with none but pages that exist, whose rows of a copy lie in one page (RUNS).
        auto fetch_plain = [&](int i) __attribute__((always_inline)) {
            if constexpr (!RUNS) fetch(i);
            else
#pragma unroll
                for (int c = 0; c < CP; c++) id[c] = table[div_by(key_of(i) + CR * (4 * c + wave), p.S)];
        };
        auto issue_plain = [&](int i, u32 st) __attribute__((always_inline)) {
            if constexpr (!RUNS) issue(i, st);
            else
#pragma unroll
                for (int c = 0; c < CP; c++) {
                    const int r = CR * (4 * c + wave), key = key_of(i) + r, kr = key - div_by(key, p.S) * (int)p.S.d;
                    const u32 page = (u32)uniform(id[c]);
                    dma16(uniform(kbase + row_at(page, p.kpp, kr, p.kpr)), k_off, smem + st + r * ROW);
                    dma16(uniform(vbase + row_at(page, p.vpp, kr, p.vpr)), v_off, smem + L::V + st + r * ROW);
                }
        };
        bool holes = false;  // whether the cache lacks any page of the run's part
        if (n > 0) {
            int first[CP];
            fetch(0);
#pragma unroll
            for (int c = 0; c < CP; c++) first[c] = id[c];
            fetch(min(1, n - 1));
            int second[CP];
#pragma unroll
            for (int c = 0; c < CP; c++) second[c] = id[c], id[c] = first[c];
            issue(0, 0);
#pragma unroll
            for (int c = 0; c < CP; c++) id[c] = second[c];
            if (n > 1) issue(1, L::TILE);
            if (n > 2) fetch(2);
            const int e1 = div_by(min(key_first + n * UK, w.hi) - 1, p.S);
            bool hole = false;
            for (int e = div_by(key_first, p.S) + (int)threadIdx.x; e <= e1; e += 256) hole |= (u32)table[e] >= (u32)p.P;
            hole = __any(hole);
            if (lane_again() == 0) flags[wave] = hole;
        }

        f16v o[DT];
#pragma unroll
        for (int d = 0; d < DT; d++) o[d] = (f16v){};
        float m = LEAST, l = 0.f, l_old = 0.f;

        if (!active) {  // no rows: the wave copies its part
            if (n > 0) {
                wait_copies();
                __syncthreads();
            }
            for (int i = 0; i < n; i++) {
                if (i + 2 < n) {
                    issue(i + 2, (u32)((i + 2) % 3 * L::TILE));
                    if (i + 3 < n) fetch(i + 3);
                }
                wait_copies();
                __syncthreads();
            }
        } else {
            // Q as the B operand of S^T = K Q^T.
            u4v qf[KS];
            float slope = 0.f;
            int pos = 0;
            {
                const int row = min(wr0 + lq, w.r1), token = div_by(row, p.G), head = run.kvh * (int)p.G.d + row - token * (int)p.G.d;
                const T* src = (const T*)p.q + (long)(w.first + token) * p.sqt + head * p.sqh;
#pragma unroll
                for (int x = 0; x < KS; x++) qf[x] = *(const u4v*)(src + (2 * x + g) * 8);
#pragma unroll
                for (int x = 0; x < KS; x++) asm volatile("" : "+v"(qf[x]));  // the loads complete here, not inside the tile loop
                if constexpr (MOD) {
                    if (p.slopes) slope = p.slopes[head] * LOG2E;
                    pos = w.p0 + token;
                }
            }
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
                    acc = product32<T>(ka[x % (KS / 2)], qf[x], acc);
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
            // What x is times in the softmax's exponent. Capped scores without a bias stay the -1 / (1 + 2^e) of their tanh (see capped), times 2 cap: that
            // a row's scores are all cap too low changes nothing. (From HIGH_CAP on, 2 cap passes 4096 and they are made whole first, as large scores
            // are, below.)
            const float scale = !MOD ? p.scale : p.cap > 0.f && !p.slopes && p.cap < HIGH_CAP ? 2.f * p.cap : 1.f;
            auto bias = [&](float (&x)[16], int key0) __attribute__((always_inline)) {
                if constexpr (MOD) {
                    if (__builtin_expect(p.cap >= HIGH_CAP, 0)) {
#pragma unroll
                        for (int r = 0; r < 16; r++) x[r] = capped<true>(x[r] * p.scale, p.cap);
                    } else if (p.cap > 0.f) {
#pragma unroll
                        for (int r = 0; r < 16; r++) x[r] = __builtin_amdgcn_rcpf(-1.f - __builtin_amdgcn_exp2f(x[r] * p.scale));
                        if (scale != 1.f) return;
#pragma unroll
                        for (int r = 0; r < 16; r++) x[r] = __builtin_fmaf(2.f * p.cap, x[r], p.cap);
                    } else {
#pragma unroll
                        for (int r = 0; r < 16; r++) x[r] *= p.scale;
                    }
                    if (p.slopes) {
                        const float d0 = (float)(pos - key0 - 4 * g);
#pragma unroll
                        for (int r = 0; r < 16; r++) x[r] = __builtin_fmaf(-slope, fabsf(d0 - (float)(8 * (r >> 2) + (r & 3))), x[r]);
                    }
                }
            };
            u4v pf[2];  // P of the two 16-key steps
            // Part k (of eight) of the P of scores x: registers 2 k, 2 k + 1.
            auto exps_into = [&](const float (&x)[16], int k, u4v& d, float by) __attribute__((always_inline)) {
                const float a = __builtin_amdgcn_exp2f(__builtin_fmaf(x[2 * k], by, -m)), b = __builtin_amdgcn_exp2f(__builtin_fmaf(x[2 * k + 1], by, -m));
                const u32 word = pair_of<T>(a, b);
                l = add_pair<T>(word, l);
                d[k & 3] = word;
            };
            auto exps = [&](const float (&x)[16], int k, float by) __attribute__((always_inline)) { exps_into(x, k, pf[k >> 2], by); };
            auto exps_to = [&](const float (&x)[16], int k, u4v& d) __attribute__((always_inline)) {
                exps_into(x, k, d, scale);
                asm volatile("" : "+v"(d), "+v"(l));
            };
            auto no_hook = [](int) {};
            // m moves only where a row's maximum of a tile exceeds it by more than 2: a lane's 16 values of P then add up to at most 64 (2^LIFT), which
            // full steps (below) look for. (With more than 8, as in the rows kernel, rows whose first keys score low went on at 6 to 8 above m, and
            // took each tile twice: 2 x 4096 in a window of 2048, whose rows begin with few keys, ran half of its workgroups at half speed.)
            auto move_max = [&](const float (&x)[16], float by) __attribute__((always_inline)) {
                float mx = x[0];
#pragma unroll
                for (int r = 1; r < 16; r++) mx = fmaxf(mx, x[r]);
                const f2 h = both_halves(mx);
                mx = fmaxf(h[0], h[1]) * by;
                if (__any(mx > m + (2.f + LIFT))) {
                    const float mn = fmaxf(m, mx - LIFT), a = __builtin_amdgcn_exp2f(m - mn);
                    m = mn;
                    l *= a;
#pragma unroll
                    for (int d = 0; d < DT; d++) o[d] *= a;
                }
            };
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
                    o[d] = product32<T>(va[d], pf[0], o[d]);
                    va[d] = read_v(vb, 1, d);
                    hook(d);
                    __builtin_amdgcn_sched_barrier(0);
                }
#pragma unroll
                for (int d = 0; d < DT; d++) {
                    o[d] = product32<T>(va[d], pf[1], o[d]);
                    hook(DT + d);
                    __builtin_amdgcn_sched_barrier(0);
                }
            };

            // Tiles all of whose keys all of the wave's rows see: full0 .. full1 - 1; tiles of the run without an end: .. ends - 1.
            int full0 = 0, full1 = 0;
            const int ends = min(n, (w.hi - key_first) / UK);

            // A tile's first part, wherever it lies: its scores, masked where not every row sees every key, the maximum, and the first half of P;
            // and its second, with one look at values that only some rows see.
            // x scale - m in one rounding is off by half a step of x scale: nothing for scores of attention, but 2^(x scale - m) would leave fp32's range
            // where scores pass 2^24. A wave that meets one of 4096 or more scales its scores first from then on, and takes no full steps.
            float sa[16], sb[16], by = scale;
            bool large = false;
            auto begin_tile = [&](int i, u32 st, u32 seen, bool masked) __attribute__((always_inline)) {
                qk(st, sa, no_hook);
                bias(sa, key_of(i));
                if constexpr (!MOD) {
                    if (!large) {
                        float a = 0.f;
#pragma unroll
                        for (int r = 0; r < 16; r++) a = fmaxf(a, fabsf(sa[r]));
                        large = __any(a * scale >= 4096.f);
                        by = large ? 1.f : scale;
                    }
                    if (__builtin_expect(large, 0))
#pragma unroll
                        for (int r = 0; r < 16; r++) sa[r] *= scale;
                }
                if (masked) {
                    const u32 mine = seen >> (4 * (lane_again() >> 5));  // register r: key 8 (r / 4) + 4 g + r % 4
#pragma unroll
                    for (int r = 0; r < 16; r++) sa[r] = mine >> (8 * (r >> 2) + (r & 3)) & 1 ? sa[r] : -__builtin_inff();
                }
                move_max(sa, by);
                l_old = l;
#pragma unroll
                for (int k = 0; k < 4; k++) exps(sa, k, by);
            };
            auto end_tile = [&](u32 st, u32 seen, bool masked) __attribute__((always_inline)) {
                if (masked) {
                    // Values that are not finite, of keys that only some rows see: key by key.
                    typedef unsigned short us2 __attribute__((ext_vector_type(2)));
                    constexpr unsigned short E = std::is_same<T, half_t>::value ? 0x7c00 : 0x7f80;
                    us2 most = {0, 0};
#pragma unroll
                    for (int x = 0; x < L::TILE / 1024; x++) {
                        const u4v v = lds_u4(smem_u + L::V + st + x * 1024 + lane_again() * 16) & 0x7fff7fffu;
#pragma unroll
                        for (int e = 0; e < 4; e++) {
                            const u32 word = v[e];
                            most = __builtin_elementwise_max(most, __builtin_bit_cast(us2, word));
                        }
                    }
                    const bool odd = most[0] >= E || most[1] >= E;
                    if (__builtin_expect(__any(odd), 0)) {
#pragma unroll
                        for (int j = 0; j < 2; j++)
#pragma unroll
                            for (int d = 0; d < DT; d++) {
                                const u4v v = read_v(v_base + st, j, d);
#pragma unroll 1
                                for (int kk = 0; kk < 16; kk++) {  // value (kk & 3) + kk / 8 x 4 of the lanes with g = kk / 4 & 1
                                    const int e0 = (kk >> 3) * 4 + (kk & 3);
                                    u4v one;
#pragma unroll
                                    for (int e = 0; e < 4; e++) one[e] = (kk >> 2 & 1) == (lane_again() >> 5) && e0 >> 1 == e ? v[e] & (kk & 1 ? 0xffff0000u : 0xffffu) : 0;
                                    const f16v x = product32<T>(one, pf[j], (f16v){});
                                    if (seen >> (16 * j + kk) & 1) o[d] += x;
                                }
                            }
                        return;
                    }
                }
                pv(st, no_hook);
            };
            // A step of the full tiles: tile i's scores are in s, its P's first half in pf[0] and l (before which l was l_old); tile i + 1 is full
            // too, and its scores go to nxt. Steps of KS (or 2 DT = KS) products: the four parts of half a tile's exponentials beside every
            // (KS / 4)-th. P is made with the m at hand: a lane's sum that grew by no more than MOST proves that no P was above it; else
            // the step ends before the product (false), and the tile is taken again by a plain step. (With the maximum moved here, O was
            // copied between registers in every step: 64 of ~300 instructions.)
            auto beside = [](int x) __attribute__((always_inline)) { return x % (KS / 4) == KS / 4 - 1; };
            auto full_step = [&](int i, u32 st, u32 st1, u32 st2, const float (&s)[16], float (&nxt)[16]) __attribute__((always_inline)) {
                if (i + 2 < ends) issue_plain(i + 2, st2);
                if (i + 3 < ends) fetch_plain(i + 3);
                qk(st1, nxt, [&](int x) { if (beside(x)) exps(s, 4 + x / (KS / 4), scale); });
                bias(nxt, key_of(i + 1));
                if (__builtin_expect(__any(!(l <= l_old + MOST)), 0)) return false;
                l_old = l;
                u4v pn;
                pv(st, [&](int x) { if (beside(x)) exps_to(nxt, x / (KS / 4), pn); });
                pf[0] = pn;
                wait_copies();
                __syncthreads();
                return true;
            };

            if (n > 0) {
                wait_copies();
                __syncthreads();
                holes = uniform(flags[0] | flags[1] | flags[2] | flags[3]) != 0;
                if (!holes) {
                    const int upto = min(w.hi, p.window > 0 ? n0 + 1 : max(n0 + 1, w.prefix));
                    full0 = first_unit_in_window<UK>(n1, p.window, key_first);
                    full1 = min(max((upto - key_first) / UK, 0), n);
                }
            }
            // Pairs of full steps i, i + 1 up to `last`: tiles .. i + 2 full, and copies of tiles without an end only (or none left to copy).
            const int last = ends == n ? full1 - 3 : min(full1 - 3, ends - 5);
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
                bool full = i >= full0 && i <= last, copied = false;  // whether tile i + 2 is on its way
                if (!full && i + 2 < n) {
                    issue(i + 2, st2);
                    if (i + 3 < n) fetch(i + 3);
                    copied = true;
                }
                if (__any(seen != 0)) {
                    while (true) {
                        begin_tile(i, st, seen, masked);
                        full = full && !large;
                        bool done = true, taken = true;  // taken: the tile's maximum is
                        while (full) {
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
                            if (!copied && i + 2 < n) {
                                issue(i + 2, st2);
                                if (i + 3 < n) fetch(i + 3);
                            }
                            copied = true;
#pragma unroll
                            for (int k = 4; k < 8; k++) exps(sa, k, by);
                            if (taken || !__any(!(l <= l_old + MOST))) break;
                        }
                        // P above the maximum at hand (a full step's look, or the last tile's after full steps): the tile again, its copies made.
                        l = l_old;
                        copied = true;
                        full = false;
                    }
                    end_tile(st, seen, masked);
                }
                i++;
                turn_stages();
                wait_copies();
                __syncthreads();
            }
        }

        // The rows turn around in LDS (chunk c of row r at c ^ (r & 15) or, of 8, c ^ (r & 7)) so that a store covers whole rows.
        if (active) {
            const int ln = lane_again(), lg = ln >> 5, lr = ln & 31;
            const f2 lh = both_halves(l);
            const float sum = lh[0] + lh[1];
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
                        const u2v word = {pair_of<T>(o[d][4 * r4] * inv, o[d][4 * r4 + 1] * inv), pair_of<T>(o[d][4 * r4 + 2] * inv, o[d][4 * r4 + 3] * inv)};
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
                            *(f4*)(turn + lr * 256 + (((8 * d + 2 * r4 + lg) ^ (lr & 15)) << 4)) = (f4){z[4 * r4], z[4 * r4 + 1], z[4 * r4 + 2], z[4 * r4 + 3]};
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
__global__ __launch_bounds__(256) void merge_kernel(PagedArgs p) { merge_parts<T, D, MT>(p); }

// ------------------------------------------------------------------------------------------------ launches

struct Plan {
    int mt, grid;
    size_t workspace;
};
static int make_plan(long T, long B, long H, long Hkv, long D, int type, Plan* plan) {
    if (T <= 0 || B <= 0 || B > MAX_SEQUENCES || Hkv <= 0 || H <= 0 || H % Hkv || (D != 64 && D != 128) || type < RDA_FP16 || type > RDA_FP32) return RDA_ERR_INVALID;
    if (T * (H / Hkv) >= 1L << 31) return RDA_ERR_INVALID;
    // Tiles of 16, 32 or 128 rows by the rows of a sequence and KV head, on average. (A lower or higher number in one of them costs time only: a chunk
    // of 512 tokens over 3584 keys beside 64 single ones over 4096 takes tiles of 32 rows, 286 us where the two alone take 75 + 197, one of 2048 over 2048
    // beside 255 of them 1017 where they take 152 + 753; beside 30 it takes tiles of 128.) us 16 / 32 / 128: 32 sequences over 4096 keys, of 16 rows 113 / 121 / 142, 32 rows 130 / 125 / 144, 64 rows 249 / 140 / 157, 96 rows
    // 368 / 324 / 172. Where all tiles of 128 rows together are few, each is cut into many parts, which cost more than the keys that
    // tiles of 32 read again: over 8192 keys, 128-row tiles x KV heads 16 (24 tokens of one sequence) 34 / 68, 32 (128 tokens) 67.7 / 66.1, 48
    // (192) 84 / 73; over 4096 keys, 32 (4 x 24 tokens) 43 / 63, 48 (2 x 96) 54 / 59, 64 (4 x 48) 70 / 61. fp32 keeps 16 rows, whose
    // matrix products bound it (32 sequences of 16 rows 186, in tiles of 32 rows 242; 32 rows 238 / 247; 512 tokens over 512 105 / 110).
    const long rows = T * (H / Hkv) / B;
    plan->mt = rows <= 16 || type == RDA_FP32 ? 16 : rows <= 64 || B * ((rows + 127) / 128) * Hkv <= 40 ? 32 : 128;
    // Two or three workgroups on each of 256 CUs, by registers: two of the tiles of 32 rows and of 128-dim ones of 16, three of 64-dim ones of 16 and of 128
    // rows (capped or biased 128-dim ones of 128: two, below). Some forms would fit one more (64-dim ones of 16 rows where pages hold whole runs, or in
    // fp32, and plain bf16 ones of 32). The workspace is sized for this grid, also where a short call launches less of it: at D = 128 in MB 8.5 for tiles
    // of 16 rows, 17 of 32, 102 of 128, half of it at D = 64 (16 rows: 6.5).
    plan->grid = (D == 128 && plan->mt == 16) || plan->mt == 32 ? 512 : 768;
    if ((T * (H / Hkv) / plan->mt + 1) * B >= 1L << 31) return RDA_ERR_INVALID;
    plan->workspace = (size_t)plan->grid * sizeof(Cut) + (size_t)plan->grid * 2 * plan->mt * (D + 2) * 4;
    return 0;
}

template <class T, int D, int MB>
static int launch_rows(const PagedArgs& a, void* stream) {
    constexpr int OP = D + 4;
    const size_t o = 4 * 16 * OP * 4, sums = (size_t)(a.B + 1) * 4, lds = o > sums ? o : sums;
    const bool mod = a.cap > 0.f || a.slopes;
    const auto launch = [&](auto kernel) { hipLaunchKernelGGL(kernel, dim3(a.grid), dim3(256), lds, (hipStream_t)stream, a); };
    if (a.S.d % RowsTile<T>::KG == 0) mod ? launch(rows_kernel<T, D, MB, true, true>) : launch(rows_kernel<T, D, MB, false, true>);
    else mod ? launch(rows_kernel<T, D, MB, true, false>) : launch(rows_kernel<T, D, MB, false, false>);
    if (const hipError_t e = hipGetLastError()) return (int)e;
    hipLaunchKernelGGL((merge_kernel<T, D, 16 * MB>), dim3(a.grid, 4 * MB), dim3(256), 0, (hipStream_t)stream, a);
    return (int)hipGetLastError();
}
template <class T, int D>
static int launch_tiles(const PagedArgs& a, void* stream) {
    const size_t lds = TilesLds<D>::BYTES;
    const auto launch = [&](auto kernel) { hipLaunchKernelGGL(kernel, dim3(a.grid), dim3(256), lds, (hipStream_t)stream, a); };
    const bool mod = a.cap > 0.f || a.slopes;
    // Rows of a copy from one scalar base: in one page, the lanes' offsets within 32 bits.
    if (a.S.d % 8 == 0 && a.kpr < 1u << 24 && a.vpr < 1u << 24) mod ? launch(tiles_kernel<T, D, true, true>) : launch(tiles_kernel<T, D, false, true>);
    else mod ? launch(tiles_kernel<T, D, true, false>) : launch(tiles_kernel<T, D, false, false>);
    if (const hipError_t e = hipGetLastError()) return (int)e;
    hipLaunchKernelGGL((merge_kernel<T, D, 128>), dim3(a.grid, 8), dim3(256), 0, (hipStream_t)stream, a);
    return (int)hipGetLastError();
}
template <class T, int D>
static int launch_paged(const PagedArgs& a, const Plan& plan, void* stream) {
    if constexpr (sizeof(T) == 2)
        if (plan.mt == 128) return launch_tiles<T, D>(a, stream);
    if constexpr (sizeof(T) == 2)
        if (plan.mt == 32) return launch_rows<T, D, 2>(a, stream);
    return launch_rows<T, D, 1>(a, stream);
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
    if ((T * (H / Hkv) / plan.mt + B) * (N * S / 32 + 1 + ahead(plan.mt, false)) >= 1L << 32) return RDA_ERR_INVALID;
    for (int i : {13, 14, 16, 17})
        if (dims[i] < 0 || dims[i] >= 1L << 32) return RDA_ERR_INVALID;
    PagedArgs a;
    a.q = q; a.o = out; a.k = k_pages; a.v = v_pages;
    a.table = table; a.starts = starts; a.lengths = lengths; a.prefix = prefix;
    a.slopes = slopes;
    a.ws = (char*)workspace;
    a.T = (int)T; a.B = (int)B; a.H = (int)H; a.Hkv = (int)Hkv; a.P = (int)P; a.N = (int)N; a.capacity = (int)(N * S);
    a.S = make_div((int)S); a.G = make_div((int)(H / Hkv));
    a.pitch = dims[6];
    a.sqt = dims[9]; a.sqh = dims[10]; a.sot = dims[11]; a.soh = dims[12];
    a.kpp = (u32)dims[13]; a.kpr = (u32)dims[14]; a.kph = dims[15]; a.vpp = (u32)dims[16]; a.vpr = (u32)dims[17]; a.vph = dims[18];
    a.scale = softcap > 0.f ? scale / softcap * 2.f * LOG2E : scale * LOG2E;
    a.cap = softcap * LOG2E;
    // Normal, positive and finite: masked scores are -inf before they meet the scale.
    if (!(a.scale >= 1.2e-38f && a.scale <= 3e38f && a.cap <= 3e38f)) return RDA_ERR_INVALID;
    a.window = window;
    // No more workgroups than units there can be: a short table of few sequences needs none that finds no work.
    const long least = plan.mt == 128 ? 32 : type == RDA_FP32 ? 64 : 128, units = (T * (H / Hkv) / plan.mt + B) * ((N * S + least - 1) / least + ahead(plan.mt, false)) * Hkv;
    const int most = plan.mt == 128 && D == 128 && (softcap > 0.f || slopes) ? 512 : plan.grid;  // that kernel's registers leave two workgroups to a CU
    a.grid = (int)(units < most ? units : most);
    a.runs = make_div(a.grid);
    a.fill = fill;
    const auto heads = [&](auto x) {
        using X = decltype(x);
        return D == 64 ? launch_paged<X, 64>(a, plan, stream) : launch_paged<X, 128>(a, plan, stream);
    };
    return type == RDA_FP16 ? heads(half_t{}) : type == RDA_BF16 ? heads(bf16_t{}) : heads(float{});
}

}  // extern "C"
