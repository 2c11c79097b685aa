"""The keys that the tiles of paged attention walk (make_tile in csrc/paged_work.h, its own text compiled with the host g++) against the keys that their rows
see: each of these once and none twice, whatever the length, the table's capacity, the window and the prefix; and the units that are taken without a mask: all
of whose keys all rows see."""
import os
import re
import shutil
import subprocess

import pytest

CSRC = os.path.join(os.path.dirname(os.path.abspath(__file__)), "..", "comfyui-rdna2-attention_amd", "csrc")

SHIM = r"""
#include <algorithm>
#include <cstdio>
#include <cstdlib>
#include <random>
#include <vector>
using std::max;
using std::min;
#define __device__
#define __forceinline__ inline
struct Div { int d; };
static int div_by(int n, const Div& v) { return n / v.d; }
struct PagedArgs {
    const int *starts, *lengths, *prefix;
    int T, capacity, window;
    Div G;
};
"""

CHECK = r"""
static std::mt19937_64 rng(1);
static long upto(long n) { return (long)(rng() % (unsigned long)(n + 1)); }
static long spread(long n) {  // small numbers as often as large ones
    long x = upto(n);
    for (long r = upto(3); r > 0; r--) x = upto(x);
    return x;
}
static long bad = 0, capped = 0, skipped = 0;

// Tiles of 128 rows take units full0 .. full1 - 1 without a mask, as the kernels have them for each of their waves of 32 rows.
template <int MT, int UK, int AHEAD, bool SKIP>
static void walk(const PagedArgs& p, int group) {
    int first;
    const int rows = seq_rows(p, 0, first);
    for (int j = 0; j * MT < rows; j++) {
        const WorkTile t = make_tile<MT, UK, AHEAD, SKIP>(p, 0, j);
        const int n = t.hi > t.lo ? t.units - AHEAD : 0;
        auto key_of = [&](int i) { return t.lo + (long)i * UK + (i >= t.head ? t.skip : 0); };
        std::vector<int> walked(t.hi + 1, 0);
        for (int i = 0; i < n; i++)
            for (long k = key_of(i); k < min(key_of(i) + UK, (long)t.hi); k++) {
                if (k < 0) { printf("key %ld\n", k); exit(1); }
                walked[k]++;
            }
        auto sees = [&](int row, int key) {
            const int at = t.p0 + row / group;
            return (key <= at && (p.window <= 0 || at - key < p.window)) || key < t.prefix;
        };
        bool wrong = n > 0 && key_of(n - 1) + UK > t.keys + 2L * UK;  // starts far behind the keys
        const int ends[] = {t.r0, t.r1};
        for (int k = 0; k < t.keys && !wrong; k++) {
            const bool seen = sees(ends[0], k) || sees(ends[1], k) || (p.window > 0 && k > t.p0 + t.r0 / group && k <= t.p0 + t.r1 / group);
            wrong = seen ? k >= t.hi || walked[k] != 1 : k < t.hi && walked[k] > 1;
        }
        if (MT == 128)
            for (int w0 = t.r0; w0 <= t.r1 && n > 0 && !wrong; w0 += 32) {
                const int w1 = min(w0 + 31, t.r1), n0 = t.p0 + w0 / group, n1 = t.p0 + w1 / group, seen_to = min(t.hi, p.window > 0 ? n0 + 1 : max(n0 + 1, t.prefix));
                const int window_first = t.lo + t.skip;
                int full0 = first_unit_in_window<UK>(n1, p.window, window_first);
                if (t.skip) full0 = max(full0, t.head);
                const int full1 = min(max((seen_to - window_first) / UK, 0), n);
                for (int i = full0; i < full1; i++)
                    for (long k = key_of(i); k < key_of(i) + UK; k++) wrong |= !sees(w0, (int)k) || !sees(w1, (int)k) || k >= t.hi;
            }
        skipped += t.skip > 0;
        if (wrong && !bad++)
            printf("length %d capacity %d window %d prefix %d rows %d tile %d of %d rows, %d keys a unit, skip %d: lo %d hi %d head %d skip %d units %d\n", p.lengths[0], p.capacity,
                   p.window, t.prefix, rows, j, MT, UK, (int)SKIP, t.lo, t.hi, t.head, t.skip, t.units);
    }
}
int main() {
    for (int i = 0; i < 40000; i++) {
        const int group = 1 + (int)upto(4), tokens = 1 + (int)spread(140), page = 16 << upto(3);
        int capacity = page * (1 + (int)spread(3000 / page)), length = (int)spread(4200), prefix = (int)spread(3000), starts[] = {0, tokens};
        if (i % 50 == 0) length = 0x7fffffff - (int)spread(5000);
        PagedArgs p = {starts, &length, upto(3) ? &prefix : nullptr, tokens, capacity, upto(3) ? (int)spread(4000) : 0, {group}};
        if (i % 50 == 0 && upto(1)) p.window = max(length - (int)spread(4000), 1);
        if (i % 97 == 0) p.window = 0x7fffffff;
        capped += length > capacity;
        walk<16, 256, 1, true>(p, group);
        walk<32, 128, 1, true>(p, group);
        walk<128, 32, 8, true>(p, group);
        walk<128, 32, 4, true>(p, group);
        walk<16, 256, 1, false>(p, group);
        walk<128, 32, 8, false>(p, group);
    }
    printf("%ld wrong tiles; %ld calls past their table, %ld tiles that leave keys out\n", bad, capped, skipped);
    return bad || capped < 5000 || skipped < 5000;
}
"""


@pytest.mark.skipif(shutil.which("g++") is None, reason="needs g++")
def test_every_visible_key_is_walked_once(tmp_path):
    text = open(os.path.join(CSRC, "paged_work.h")).read()
    struct, = re.findall(r"^struct WorkTile \{\n.*?^\};\n", text, re.M | re.S)
    rows, = re.findall(r"^__device__ __forceinline__ int seq_rows\(.*?^\}\n", text, re.M | re.S)
    tile, = re.findall(r"^template <int MT, int UK, int AHEAD, bool SKIP = false>\n__device__ __forceinline__ WorkTile make_tile\(.*?^\}\n", text, re.M | re.S)
    full, = re.findall(r"^template <int UK>\n__device__ __forceinline__ int first_unit_in_window\(.*?^\}\n", text, re.M | re.S)
    source, exe = tmp_path / "walk.cpp", tmp_path / "walk"
    source.write_text(SHIM + struct + rows + tile + full + CHECK)
    subprocess.run(["g++", "-std=c++17", "-O2", "-fwrapv", str(source), "-o", str(exe)], check=True)
    r = subprocess.run([str(exe)], capture_output=True, text=True, timeout=600)
    assert r.returncode == 0, r.stdout
