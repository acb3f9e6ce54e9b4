"""Whatever a plan of paged_attention_shared needs, the call has: work-groups,
room for partial results, entries of the map of tokens (CPU only).

The host knows sizes, not lengths, and takes bounds of what the plan, on the
device, comes to from the lengths.  The bounds are the library's own, compiled for
the host from its source; the plan's counts are formed again here, for every number
of parts that it may take.
"""

from __future__ import annotations

import random
import shutil
import subprocess
from pathlib import Path

import pytest

CSRC = Path(__file__).resolve().parents[1] / "kda-ascendc_amd" / "csrc"
HIPCC = next((x for x in ("/opt/rocm/bin/hipcc", shutil.which("hipcc")) if x and Path(x).exists()), None)

PROGRAM = r"""
#include "kda_paged_shared.hip"
#include <cstdio>
using namespace kda;
int main() {
    printf("%d %d %d %d %d %d %d %d\n", MT, WIDE_MT, WIDE, ROWS, IN_JOIN, FEW_PARTS, Shape<MANY>::SLOTS, Shape<MANY>::LEAST);
    long long N, T, HQ, HKV, M, NG, page;
    int packed, D, offsets = 0;
    while (scanf("%lld %lld %lld %lld %lld %lld %lld %d %d", &N, &T, &HQ, &HKV, &M, &page, &NG, &packed, &D) == 9) {
        SharedParams p{};
        p.N = N, p.T = T, p.HQ = HQ, p.HKV = HKV, p.G = HQ / HKV, p.M = M, p.NG = NG, p.causal = 1;
        p.page_shift = __builtin_ctzll(page);
        p.cu_seqlens = packed ? &offsets : nullptr;
        printf("%d %lld %lld %lld %d %d\n", together(p, D), (long long)room_of(p), (long long)units_of(p),
               (long long)sharing_tokens(p), rounds_of(p), few_only(p));
    }
}
"""


class Constants:
    def __init__(self, text):
        (self.MT, self.WIDE_MT, self.WIDE, self.ROWS, self.IN_JOIN, self.FEW_PARTS, self.SLOTS, self.LEAST) = map(int, text.split())


@pytest.fixture(scope="module")
def host_sizes(tmp_path_factory):
    """(constants, the bounds of each of some calls)."""
    if HIPCC is None:
        pytest.skip("no hipcc")
    path = tmp_path_factory.mktemp("sizes")
    (path / "sizes.hip").write_text(PROGRAM)
    # (host code only: there are no kernels to link, and none is launched)
    subprocess.run([HIPCC, "--offload-host-only", "-std=c++17", "-O1", "-Wl,--unresolved-symbols=ignore-all", f"-I{CSRC}",
                    str(path / "sizes.hip"), "-o", str(path / "sizes")], check=True, capture_output=True)

    def run(calls):
        text = "\n".join(" ".join(str(int(x)) for x in c) for c in calls) + "\n"
        lines = subprocess.run([str(path / "sizes")], input=text, check=True, capture_output=True, text=True).stdout.splitlines()
        assert len(lines) == len(calls) + 1
        return Constants(lines[0]), [tuple(map(int, x.split())) for x in lines[1:]]

    return run


def ceil(a, b):
    return -(-a // b)


def needs(c, call, groups, new, lens, rounds, few_only):
    """(units, room in 4 rows, sharing tokens, what it came by) of a plan, the most
    over the numbers of parts that it may take."""
    N, T, HQ, HKV, M, page, NG, packed, D = call
    G = HQ // HKV
    shares = [-1] * N
    for g, (a, b, shared) in enumerate(groups):
        for n in range(a, b):
            if shared > 0 and 0 < new[n] and new[n] * G < c.MT and lens[n] - new[n] >= shared:
                shares[n] = g
    count = [shares.count(g) for g in range(NG)]
    shares = [g if g >= 0 and count[g] >= 2 else -1 for g in shares]
    records = [(sum(new[n] for n in range(a, b) if shares[n] == g), shared, 0, True, -1) for g, (a, b, shared) in enumerate(groups)]
    records += [(new[n], lens[n], groups[g][2] if (g := shares[n]) >= 0 else 0, False, g) for n in range(N)]
    few_tiles = few_records = many = many_tiles = 0
    work = []
    for tokens, keys, start, group, of in records:
        if tokens == 0:
            continue
        rows = tokens * G
        few = rows <= c.ROWS
        keys_a_tile, tile = (32, c.ROWS) if few else (64, c.MT)
        tiles = max(1, ceil(keys, keys_a_tile) - start // keys_a_tile)
        mt = ceil(rows, tile)
        if few and of >= 0 and tiles <= c.IN_JOIN:
            continue
        work.append((rows, few, tiles, mt, group, of))
        if few:
            few_records += HKV
            few_tiles += tiles * HKV
        else:
            many += mt * HKV
            many_tiles += mt * HKV * tiles
    waves = 4 if few_only else 8
    slots, fine = 2048 // waves, 4 * waves * (128 // D)
    size = max(waves, ceil(few_tiles, c.FEW_PARTS), min(ceil(few_tiles, slots), fine))
    wide = many >= c.WIDE
    units = many // 2 if wide else many
    beside = few_tiles // size + few_records
    takes = [r * c.SLOTS - (beside if beside <= c.SLOTS // 4 else 0) for r in range(1, rounds + 1)]
    takes = [0] + [x for x in takes if 0 < units <= x]
    most_units = most_room = 0
    by = set()
    if few_tiles > slots * size:
        by.add("more parts of few rows than run at once")
    for share in takes:
        all_units = all_room = 0
        for rows, few, tiles, mt, group, of in work:
            if few:
                parts = ceil(tiles, size)
            else:
                own, parts = share, 1
                if wide and not group:
                    narrow, mt = mt, (mt + 1) // 2
                    own = 2 * share - (ceil(share, mt) if narrow % 2 else 0)
                    by.add("row tiles of 256")
                    if of >= 0:
                        by.add("row tiles of 256 that share")
                if share > 0:
                    parts = max(1, min(tiles // c.LEAST, int(tiles * own / many_tiles)))
                if parts > 1:
                    by.add("many rows' keys cut")
            all_units += mt * parts * HKV
            if parts > 1 or group or of >= 0:
                all_room += ceil(rows, 4) * parts * HKV
        most_units, most_room = max(most_units, all_units), max(most_room, all_room)
    if any(not few and of >= 0 for _, few, _, _, _, of in work):
        by.add("many rows that share")
    return most_units, most_room, sum(new[n] for n in range(N) if shares[n] >= 0), by


def draw(rng):
    """A call of any sizes, and its lengths."""
    N = rng.choice([2, 3, 5, 8, 17, 64, 130, 300, 700])
    G = rng.choice([1, 2, 3, 4, 5, 7, 8, 16, 35, 64, 130])
    HKV = rng.choice([1, 2, 4, 8, 32])
    D = rng.choice([64, 128])
    packed = rng.random() < 0.6
    if packed:
        most = rng.choice([1, 2, 40, 127 // G + 1, 300, 2000])
        new = [rng.choice([0, 1, 1, rng.randint(0, most)]) for _ in range(N)]
        T = max(1, sum(new)) + rng.choice([0, 0, 9])
    else:
        T = rng.choice([1, 1, 2, 3, 8, 16, 40, max(1, 128 // G), max(1, 32 // G)])
        new = [T] * N
    cuts = sorted(rng.randint(0, N) for _ in range(rng.choice([2, 2, 3, 5, 9]))) if rng.random() < 0.7 else list(range(0, N + 1, 2))
    longest = rng.choice([40, 700, 5000, 16000, 100000])
    groups = [(a, b, rng.choice([0, 1, rng.randint(1, longest), longest])) for a, b in zip(cuts, cuts[1:])]
    lens = [0] * N
    for a, b, shared in groups:
        lens[a:b] = [shared] * (b - a)
    own = rng.choice([0, 50, 600, 5000, 50000])
    lens = [x + new[n] + rng.randint(0, own) if rng.random() < 0.97 else rng.choice([0, 1, new[n] // 2]) for n, x in enumerate(lens)]
    page = rng.choice([16, 64, 1024])
    M = max(ceil(max(lens), page), ceil(230 << 20, page * HKV * D * 4 * N), 1)
    return (N, T, G * HKV, HKV, M, page, len(groups), packed, D), groups, new, lens


def test_a_plan_fits(host_sizes):
    rng = random.Random(5)
    cases = [draw(rng) for _ in range(6000)]
    # 32 pairs behind 9000 tokens; chunks beside sequences of 33 to 127 rows that share; all of a sequence's rows in one tile more
    cases.append(((64, 1, 32, 8, 600, 16, 32, 0, 128), [(2 * g, 2 * g + 2, 9000) for g in range(32)], [1] * 64, [9100] * 64))
    new = [20, 31, 12, 9, 400, 700, 900]
    cases.append(((7, sum(new), 128, 32, 2000, 16, 1, 1, 128), [(0, 7, 6000)], new, [6000 + x for x in new]))
    seen, worst = set(), [0.0, 0.0, 0.0]
    constants, bounds = host_sizes([x[0] for x in cases])
    done = 0
    for (call, groups, new, lens), (together, room, units, entries, rounds, few_only) in zip(cases, bounds):
        if not together:
            continue
        done += 1
        got_units, got_room, sharing, by = needs(constants, call, groups, new, lens, rounds, few_only)
        assert got_units <= units and got_room <= room and sharing <= entries, (call, groups, new, lens)
        seen |= by
        worst = [max(w, x) for w, x in zip(worst, (got_units / units, got_room / room, sharing / entries))]
    assert done > 3000 and len(seen) == 5, (done, seen)
    # (the bounds are of use: some call comes near to each)
    assert min(worst) > 0.5, worst
