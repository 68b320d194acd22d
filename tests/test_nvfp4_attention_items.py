"""What packed_attention_nvfp4 deals its work into: the workspace holds the items of any lengths that a call's sizes allow, and is
not much larger than what some of them need. The lengths are known to the device alone; here its numbering is restated."""

import random

import pytest

from appcorr_amd import _lib


def shape(rows, S, Hq, Hk, Dh, cap):
    """Rows and keys of a tile, parts aimed at (0: keys are not split) and the fewest key tiles of a part, by the call's sizes."""
    G, seqs = Hq // Hk, max(1, min(S, rows))
    mean = -(-rows * G // seqs)
    R = 16 if mean <= 32 else 256 if Dh == 128 and mean > 192 else 128
    tiles = max(rows * G // R, seqs)
    split = tiles * Hk < 4 * 256 and cap > 2048
    target = -(-{16: 4, 128: 2, 256: 1}[R] * 256 // Hk) if split else 0
    return R, 128 if R == 16 else 64, target, 2 if R == 16 else 6


def items(nq, nk, G, R, KT, target, min_tiles):
    """Items of a key head with these rows and keys: tiles of rows times parts of keys."""
    tiles = [(-(-m * G // R), -(-n // KT)) for m, n in zip(nq, nk)]
    chunk = max(min_tiles, -(-sum(t * k for t, k in tiles) // target))
    return sum(t * max(1, (2 * k + chunk) // (2 * chunk)) for t, k in tiles)


def lengths(r, rows, S, cap):
    """Rows and keys of S sequences, of all kinds: as many rows as there are, or fewer."""
    kind = r.randrange(6)
    nq = [0] * S
    if kind == 0:  # all in one
        nq[r.randrange(S)] = rows
    elif kind == 1:  # even
        nq = [rows // S + (i < rows % S) for i in range(S)]
    else:
        cuts = sorted(r.randint(0, rows) for _ in range(S - 1))
        nq = [b - a for a, b in zip([0, *cuts], [*cuts, rows])]
    if kind == 2:  # one token each but for one
        nq = [1] * min(S, rows) + [0] * (S - min(S, rows))
        nq[0] += rows - sum(nq)
    nk = [cap if kind < 3 else r.randint(0, cap) if kind == 3 else int(cap ** r.random()) for _ in range(S)]
    if kind == 5:  # lengths that round up to a further part
        base = r.randint(1, cap)
        nk = [min(cap, base * r.choice((1, 3, 5)) // 2) for _ in range(S)]
    return nq, nk


CASES = [(1, 1, 8, 8, 64, 4096), (4, 4, 32, 8, 128, 16385), (32, 32, 32, 8, 128, 16385), (64, 32, 16, 16, 64, 8192),
         (512, 3, 32, 8, 128, 8704), (700, 3, 16, 16, 64, 9000), (2048, 8, 32, 8, 128, 8192), (100, 70, 4, 1, 64, 4000),
         (300, 300, 4, 1, 64, 2500), (17, 5, 6, 2, 128, 2049), (1, 1, 64, 64, 128, 1 << 20), (5, 9, 1, 1, 64, 100000)]


@pytest.mark.parametrize("rows,S,Hq,Hk,Dh,cap", CASES)
def test_the_workspace_holds_any_lengths(rows, S, Hq, Hk, Dh, cap):
    R, KT, target, least = shape(rows, S, Hq, Hk, Dh, cap)
    elems = _lib.load().oudjat_packed_attention_nvfp4_workspace_elems(rows, S, Hq, Hk, Dh, cap)
    assert target and elems > 0
    held, rest = divmod(elems, Hk * (R * (Dh + 2) + 4))  # a reference, a sum and R rows of Dh; four ints for the merge
    assert rest == 0
    r = random.Random(rows + cap)
    most = max(items(*lengths(r, rows, S, cap), Hq // Hk, R, KT, target, least) for _ in range(3000))
    assert most <= held
    assert held <= 3 * most + 8


@pytest.mark.parametrize("rows,S,Hq,Hk,Dh,cap", [
    (4, 4, 32, 8, 128, 2048), (2048, 2, 16, 16, 64, 2048), (65536, 8, 32, 8, 128, 8192), (2000, 2000, 8, 2, 64, 4096)])
def test_calls_that_do_not_split_need_no_workspace(rows, S, Hq, Hk, Dh, cap):
    assert shape(rows, S, Hq, Hk, Dh, cap)[2] == 0
    assert _lib.load().oudjat_packed_attention_nvfp4_workspace_elems(rows, S, Hq, Hk, Dh, cap) == 0
