"""How the paged attention's CTAs share the blocks of a call (csrc/paged_attention.cuh), walked on the CPU with the kernel's own arithmetic: every block once, every part
where the adding CTA looks for it, counters at zero behind the call.  And the same where CTAs read different lengths, which a caller that changes them too
early brings about: no index leaves its array, the call ends, its counters are zero, and it says so if a row's parts did not come together."""
import ctypes as C
import os
import shutil
import subprocess

import numpy as np
import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
SRC = r"""
#include <map>
#include <unordered_set>
#include <vector>
#include "%s/zklm_compile_b200/csrc/paged_attention.cuh"
using namespace zkb;

struct Call { u32 num_seqs, kv_heads, slices, ctas, block; u64 positions; };

// What a CTA makes of the lengths that it read: as in the kernel, one lane for the warp.
struct Share { bool aligned; u64 per, from, to, total; };
static Share share_of(const Call& c, const int* lens, u32 cta) {
    const u32 grps = c.kv_heads * c.slices;
    u64 total = 0, rows = 0;
    u32 len;
    for (u32 s = 0; s < c.num_seqs; s++) { const u32 nb = pa_blocks(c.positions, lens[s], c.block, len); total += nb; rows += nb != 0; }
    Share r{false, 0, 0, 0, total * grps};
    r.per = (r.total + c.ctas - 1) / c.ctas;
    if (c.num_seqs <= PA_FEW && rows && rows * grps <= c.ctas)
        for (u32 more = 0; more < 3 && !r.aligned; more++) {
            const u32 p = (u32)r.per + (more ? ((u32)r.per + 7) / 8 * more : 0);
            u64 shares = 0;
            for (u32 s = 0; s < c.num_seqs; s++) shares += (pa_blocks(c.positions, lens[s], c.block, len) + p - 1) / p;
            if (shares * grps <= c.ctas) { r.aligned = true; r.per = p; r.total = shares * grps; }
        }
    r.from = r.aligned ? cta : r.per * cta;
    r.to = r.aligned ? (r.from < r.total ? r.from + 1 : r.from) : r.from + r.per < r.total ? r.from + r.per : r.total;
    return r;
}

// lens: [ctas][versions][num_seqs], what each CTA reads when it counts, when it looks for its share and when it steps on (the same one for up to PA_FEW sequences,
// which are read once).  Returns 0, or the line of the check that failed.  *outcome: bit 0: a next call is told that parts are left over, bit 1: this one that blocks
// are missing.
#define CHECK(x) do { if (!(x)) return __LINE__; } while (0)
extern "C" int walk(u32 num_seqs, u32 kv_heads, u32 slices, u32 ctas, u32 block, u64 positions, const int* lens, u32 versions, int same, int* outcome) {
    const Call c{num_seqs, kv_heads, slices, ctas, block, positions};
    const u32 grps = kv_heads * slices;
    const bool few = num_seqs <= PA_FEW;
    std::vector<u32> arrived(ctas, 0);
    std::unordered_set<u64> blocks;                         // (sequence, item, block)
    std::map<u64, std::pair<u32, u32>> rows;                // (sequence, item) -> first CTA and parts, as each CTA sees them
    u32 begun = 0;
    *outcome = 0;
    for (u32 n = 0; n < ctas; n++) {
        const u32 cta = (n + (u32)lens[0]) %% ctas;         // in any order, here one of ctas
        const int* at[3];
        for (u32 v = 0; v < 3; v++) at[v] = lens + ((size_t)cta * versions + (few ? 0 : v %% versions)) * num_seqs;
        const Share s = share_of(c, at[0], cta);
        CHECK(!pa_stale(begun));                            // a CTA that begins is not misled by those that have begun, brought and added
        begun += pa_began(cta, ctas);
        bool gave_up = false;
        if (s.from < s.to) {
            u32 start = 0, start_len = 0;
            u64 rest = 0, before = 0;
            for (u32 q = 0; q < num_seqs; q++) {
                u32 len, nb = pa_blocks(positions, at[1][q], block, len);
                const u64 shares = s.aligned ? (nb + s.per - 1) / s.per : nb;
                if (nb && before <= s.from && s.from < before + shares * grps) { start = q; start_len = len; rest = s.from - before; }
                before += shares * grps;
            }
            PaWalk w{};
            w.nb = pa_blocks(positions, (int)start_len, block, w.len);
            if (w.nb == 0) gave_up = true;
            else w.start(start, rest, s.to - s.from, s.aligned, (u32)s.per, slices);
            PaWalk l = w;
            u64 copies = 0, used = 0;
            while (l.left) {                                // the copies' walk: a block at a time
                CHECK(l.seq < num_seqs && l.kvh < kv_heads && l.slice < slices && l.blk < l.nb);
                copies++;
                if (l.step(1, slices, kv_heads)) l.next_seq(num_seqs, positions, block, [&](u32 q) { return at[2][q]; });
            }
            while (w.left) {
                const u32 first = w.blk, count = w.left < w.nb - first ? w.left : w.nb - first;
                CHECK(w.seq < num_seqs && w.kvh < kv_heads && w.slice < slices && first < w.nb && count > 0 && (u64)w.len <= positions);
                used += count;
                const u64 item = ((u64)w.seq * kv_heads + w.kvh) * slices + w.slice;
                if (same) for (u32 b = first; b < first + count; b++) CHECK(blocks.insert(item << 32 | b).second);
                if (first || count < w.nb) {
                    const PaParts p = pa_parts(s.aligned, s.per, ctas, cta, s.to - w.left, first, w.nb);
                    CHECK(p.n >= 1 && p.first_cta < ctas && (u64)p.first_cta + p.n <= ctas);
                    if (same) {
                        CHECK((cta == p.first_cta) == (first == 0) && p.first_cta <= cta && cta < p.first_cta + p.n);
                        auto seen = rows.emplace(item, std::make_pair(p.first_cta, p.n));
                        CHECK(seen.first->second == std::make_pair(p.first_cta, p.n));
                    }
                    const bool all = arrived[p.first_cta]++ == p.n - 1;
                    if (all) arrived[p.first_cta] -= p.n;
                    begun += pa_brought(1, all ? p.n : 0);
                }
                if (w.step(count, slices, kv_heads)) {
                    w.next_seq(num_seqs, positions, block, [&](u32 q) { return at[2][q]; });
                    if (!w.left) gave_up = true;
                }
            }
            const u64 mine = s.aligned ? s.per : s.to - s.from;
            CHECK(copies <= mine && used <= mine);
            if (same) CHECK(!gave_up && copies == used && (s.aligned || used == s.to - s.from));
        }
        if (gave_up) *outcome |= 2;
    }
    CHECK((begun & 0xffffu) == 0);
    u32 rest = 0;
    for (u32 a : arrived) rest += a;
    CHECK(begun == rest << 16 && pa_stale(begun) == (rest != 0));           // the next call's first CTA sees exactly what is left
    if (rest) *outcome |= 1;
    if (same) {
        u64 total = 0;
        u32 len;
        for (u32 q = 0; q < num_seqs; q++) total += (u64)pa_blocks(positions, lens[q], block, len) * grps;
        CHECK(!begun && blocks.size() == total);
    }
    return 0;
}

extern "C" u32 halves(u32 tiles, u32 slot, u32 ns) { return pa_halves(tiles, slot, ns); }
"""


@pytest.fixture(scope="module")
def lib(tmp_path_factory):
    if not shutil.which("nvcc"):
        pytest.skip("nvcc not on PATH")
    d = tmp_path_factory.mktemp("shares")
    (d / "s.cu").write_text(SRC % ROOT)
    subprocess.run(["nvcc", "-gencode", "arch=compute_100a,code=sm_100a", "-O2", "-std=c++17", "--extended-lambda", "-Xcompiler", "-fPIC", "-shared",
                    "-o", str(d / "s.so"), str(d / "s.cu")], check=True, capture_output=True)
    return C.CDLL(str(d / "s.so"))


def batch(rng, seqs):
    kind = rng.integers(0, 5)
    if kind == 0:
        return rng.integers(0, 4000, seqs)
    if kind == 1:
        return np.where(rng.random(seqs) < 0.7, 0, rng.integers(1, 20000, seqs))
    if kind == 2:
        return rng.integers(0, 3, seqs) * 128
    if kind == 3:
        return np.full(seqs, rng.integers(1, 200000))
    return np.where(rng.random(seqs) < 0.1, rng.integers(-5, 1 << 31, seqs), rng.integers(1, 300, seqs))


def shapes(seed, n, most=(1, 2, 7, 40, 130, 256, 257, 700)):
    rng = np.random.default_rng(seed)
    for _ in range(n):
        seqs, block = int(rng.choice(most)), int(rng.choice([80, 128, 192]))
        lens = batch(rng, seqs).astype(np.int64)
        yield rng, seqs, int(rng.choice([1, 2, 3, 8, 12])), int(rng.choice([1, 1, 2, 5])), int(rng.choice([1, 3, 77, 148])), block, 1 << 18, lens


def call(lib, seqs, kv, slices, ctas, block, positions, lens, versions, same):
    told = C.c_int(0)
    lens = np.ascontiguousarray(lens, np.int32)
    assert lens.size == ctas * versions * seqs
    line = lib.walk(seqs, kv, slices, ctas, block, C.c_uint64(positions), lens.ctypes.data_as(C.c_void_p), versions, int(same), C.byref(told))
    assert line == 0, f"line {line} of the walk"
    return told.value


def test_every_block_is_taken_once(lib):
    for _, seqs, kv, slices, ctas, block, positions, lens in shapes(1, 120):
        assert call(lib, seqs, kv, slices, ctas, block, positions, np.tile(lens, (ctas, 1)), 1, True) == 0


def test_lengths_that_change_meanwhile(lib):
    """A length or all of them, by a little or to nothing, for some of the CTAs; with more than 256 sequences within a CTA too."""
    told = []
    for rng, seqs, kv, slices, ctas, block, positions, lens in shapes(2, 200):
        seen = np.tile(lens, (ctas, 3, 1))
        other = lens.copy()
        change = rng.integers(0, 4)
        where = slice(None) if change == 0 else rng.integers(0, seqs, max(1, seqs // 8))
        other[where] = {0: 0, 1: 0, 2: np.maximum(0, lens[where] - 1), 3: np.minimum((1 << 31) - 1, np.maximum(lens[where], 0) + 5000)}[int(change)]
        seen[rng.random((ctas, 3)) < rng.choice([0.05, 0.5])] = other
        told.append(call(lib, seqs, kv, slices, ctas, block, positions, seen, 3, False))
    assert {1, 2} <= set(told) and 0 in told


@pytest.mark.parametrize("ns", [2, 3, 4, 6])
def test_half_tiles_under_way(lib, ns):
    """A warp that gives up waits for the last ns of its copies; keys and values are copied in turn, and it may be between the two."""
    for n in range(3 * ns + 5):
        assert lib.halves((n + 1) // 2, n % ns, ns) == n
