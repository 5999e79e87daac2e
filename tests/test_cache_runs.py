"""How the attention over a paged cache cuts a call into runs (csrc/cache_runs.cuh), compiled for the host: every
pair of cells of every tile in one run, in order, at sizes that no test could attend to."""
import ctypes as C
import subprocess

import numpy as np
import pytest

from conftest import ROOT

SOURCE = r"""
#include <string.h>
#include "cache_runs.cuh"
using namespace lsx;

// Pairs of tile k, by its positions in 64 bits.
static long long pairs_of(const SequenceRows& s, int tokens, int k) {
    const long long last = (k + 1ll) * tokens < s.count ? (k + 1ll) * tokens : s.count;
    const long long seen = (long long)s.length - s.count + last;
    return seen <= 32 ? 1 : (seen + 31) / 32;
}

// 0 where the parts of all blocks' runs are the call's pairs in order, else what is wrong with the first that is not.
extern "C" int cut(const int* counts, const int* lengths, int sequences, int tokens, unsigned heads, int blocks, int whole) {
    long long total = 0;
    for (int b = 0; b < sequences; ++b) {
        const SequenceRows s = {b, 0, counts[b], lengths[b]};
        long long one = 0;
        for (int k = 0; k < tile_count(s, tokens); ++k) {
            if (cost_before(s, tokens, k) != one) return 1;
            one += kTileCost + pairs_of(s, tokens, k);
        }
        if (sequence_cost(s, tokens) != one) return 2;
        total += one * heads;
    }
    const long long share = (total + blocks - 1) / blocks, run = share < kLeastRun ? kLeastRun : share;
    int sequence = 0, k = 0;
    unsigned head = 0;
    long long pair = 0;  // the next part's
    for (int block = 0; block < blocks; ++block) {
        Run left = {run * block, run * (block + 1ll) < total ? run * (block + 1ll) : total, 0, 0};
        if (left.at >= left.end) break;
        long long before = 0;
        for (;; ++left.sequence) {
            const SequenceRows s = {0, 0, counts[left.sequence], lengths[left.sequence]};
            const long long cost = sequence_cost(s, tokens) * heads;
            if (left.at < before + cost) break;
            before += cost;
        }
        left.offset = left.at - before;
        while (left.at < left.end) {
            if ((int)left.sequence >= sequences) return 3;
            const SequenceRows s = {0, 0, counts[left.sequence], lengths[left.sequence]};
            const Run was = left;
            RunTile t;
            const bool some = next_tile(left, s, tokens, heads, whole, t);
            if (left.at < was.at || left.offset < 0 || (left.at == was.at && left.sequence == was.sequence)) return 4;  // no end
            if (!some) continue;
            while (sequence < sequences && counts[sequence] == 0) ++sequence;
            if ((int)left.sequence != sequence || t.head != head || t.k != k || t.first != pair) return 5;
            if (t.pairs != pairs_of(s, tokens, k) || t.last <= t.first || t.last > t.pairs) return 6;
            if (whole && (t.first != 0 || t.last != t.pairs)) return 7;
            pair = t.last;
            if (pair < t.pairs) continue;
            pair = 0;
            if (++k < tile_count(s, tokens)) continue;
            k = 0;
            if (++head < heads) continue;
            head = 0;
            ++sequence;
        }
    }
    while (sequence < sequences && counts[sequence] == 0) ++sequence;
    return sequence == sequences && head == 0 && k == 0 && pair == 0 ? 0 : 8;
}
"""


@pytest.fixture(scope="module")
def cut(tmp_path_factory):
    folder = tmp_path_factory.mktemp("runs")
    (folder / "runs.cpp").write_text(SOURCE)
    subprocess.run(["g++", "-std=c++17", "-O2", "-fwrapv", "-shared", "-fPIC", "-I", str(ROOT / "laplacesscissors_b200" / "csrc"),
                    "-o", str(folder / "runs.so"), str(folder / "runs.cpp")], check=True, timeout=300)
    call = C.CDLL(str(folder / "runs.so")).cut

    def run(counts, lengths, tokens, heads, blocks=444, whole=False):
        counts, lengths = (np.ascontiguousarray(a, np.int32) for a in (counts, lengths))
        return call(counts.ctypes.data_as(C.c_void_p), lengths.ctypes.data_as(C.c_void_p), C.c_int(len(counts)), C.c_int(tokens),
                    C.c_uint(heads), C.c_int(blocks), C.c_int(whole))
    return run


@pytest.mark.parametrize("tokens", [1, 2, 4, 8, 16])
@pytest.mark.parametrize("whole", [False, True])
def test_every_pair_once_and_in_order(cut, tokens, whole):
    rng = np.random.default_rng(tokens)
    for _ in range(60):
        n = int(rng.integers(1, 30))
        lengths = (10.0 ** rng.uniform(0, 5, n)).astype(int) * (rng.random(n) < 0.9)
        counts = np.where(rng.random(n) < 0.3, rng.integers(0, 300, n), rng.integers(0, 3, n))
        if counts.sum():
            assert cut(counts, lengths, tokens, int(rng.integers(1, 20)), int(rng.integers(1, 700)), whole) == 0


# Rows and positions whose tiles cost 2^32 and more: a prompt of 523889 rows with 16 query heads a key head, and
# shorter ones behind a million positions.
@pytest.mark.parametrize("counts,lengths,tokens,heads", [
    ([523888], [523888], 1, 2), ([523889], [523889], 1, 2), ([524889], [524889], 1, 2), ([1, 600000, 5], [9, 600000, 70], 1, 3),
    ([129060], [1129060], 1, 2), ([200000, 3], [1200000, 40], 1, 1), ([300000], [1300000], 2, 2), ([500000], [1500000], 4, 2),
    ([1100000], [1100000], 4, 1), ([1 << 20] * 2, [1 << 20] * 2, 2, 1)])
def test_long_prompts(cut, counts, lengths, tokens, heads):
    for blocks in (296, 444, 592):
        assert cut(counts, lengths, tokens, heads, blocks) == 0


# Lengths up to 2^31 - 1, whose pairs end beyond what 32 bits with a sign hold.
@pytest.mark.parametrize("tokens", [1, 2, 8, 16])
@pytest.mark.parametrize("length", [2 ** 31 - 1, 2 ** 31 - 16, 2 ** 31 - 33, 2 ** 31 - 300])
def test_lengths_at_the_end_of_their_type(cut, tokens, length):
    for counts in ([1], [100], [3000, 1, 70]):
        for blocks in (296, 444, 592):
            assert cut(counts, [length] * len(counts), tokens, 2, blocks) == 0
