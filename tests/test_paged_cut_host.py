"""CPU: the cut of an attention call's work over the GPU (Walk, csrc/paged_dev.cuh), with a warp's lanes as fibers."""
import os
import random
import re
import subprocess

import pytest

HERE = os.path.dirname(os.path.abspath(__file__))
CSRC = os.path.join(os.path.dirname(HERE), "phantom-a100_b200", "csrc")
CUDA = os.environ.get("CUDA_HOME", "/usr/local/cuda")


@pytest.fixture(scope="module")
def cut(tmp_path_factory):
    if not os.path.isdir(os.path.join(CUDA, "include")):
        pytest.skip("needs the CUDA headers")
    top = tmp_path_factory.mktemp("cut")
    src = top / "a" / "csrc"
    src.mkdir(parents=True)

    def text(*path):
        with open(os.path.join(*path)) as f:
            return f.read()

    (src / "sm100_ptx.cuh").write_text("#pragma once\n")
    for name in ("paged.h", "paged_dev.cuh"):
        (src / name).write_text(text(CSRC, name))
    (top / "include").mkdir()
    (top / "include" / "phantom_attn.h").write_text(text(CSRC, "..", "..", "include", "phantom_attn.h"))
    rows = re.search(r"template <int NT, int BN>\nstruct RowBlocks \{.*?\n\};\n", text(CSRC, "attn_paged.cu"), re.S).group()
    tokens = re.search(r"struct (?:alignas\(16\) )?TokenBlocks \{.*?\n\};\n", text(CSRC, "attn_paged_tc_sm100.cu"), re.S).group()
    (src / "blocks.h").write_text("constexpr int BN = 128;\n" + rows.replace("BN", "B_N") + tokens)
    (src / "paged_cut.cpp").write_text(text(HERE, "harness", "paged_cut.cpp"))
    exe = str(top / "cut")
    subprocess.run(["g++", "-std=c++17", "-O1", "-w", f"-I{CUDA}/include", "paged_cut.cpp", "-o", exe], cwd=src, check=True)

    def run(kind, causal, group, heads, grid, kv, cu, total=None, page=16, width=4096, changes=()):
        args = [kind, causal, group, heads, grid, page, width, cu[-1] if total is None else total, len(kv), *kv, *cu, len(changes),
                *(x for c in changes for x in c)]
        done = subprocess.run([exe, *map(str, args)], capture_output=True, text=True, timeout=60)
        assert done.returncode == 0, done.stdout[-200:] + done.stderr
        return [tuple(map(int, line.split())) for line in done.stdout.splitlines()]
    return run


def tiles(kind, causal, group, n, t, blk):
    """Tiles of block `blk` of a sequence's n new tokens over its t cached ones, by the definition; None past the last."""
    per, bn = {"rows8": (8, 64), "rows16": (16, 128), "chunk": (2 * (128 // group), 128)}[kind]
    units = n if kind == "chunk" else n * group
    if blk * per >= units:
        return None
    last = min(units, (blk + 1) * per) - 1
    last = last if kind == "chunk" else last // group
    sees = max(0, min(t, t - n + last + 1)) if causal else t
    return max(1, -(-sees // bn))


@pytest.mark.parametrize("kind", ["rows8", "rows16", "chunk"])
@pytest.mark.parametrize("seed", range(12))
def test_every_tile_is_taken_once(cut, kind, seed):
    rng = random.Random(seed)
    batch, heads, group = rng.choice([1, 2, 5, 40, 70]), rng.choice([1, 3, 8]), rng.choice([1, 4, 5, 16])
    causal, grid = rng.randint(0, 1), rng.choice([1, 7, 148])
    new = [rng.choice([0, 1, 1, 2, 9, 300] if batch < 40 else [0, 1, 1, 3]) for _ in range(batch)]
    kv = [rng.choice([0, n // 2, n, n + rng.randint(0, 5000)]) for n in new]
    cu = [sum(new[:i]) for i in range(batch + 1)]
    parts = {}
    for cta, b, h, blk, tile, cnt, nt, c0, c1 in cut(kind, causal, group, heads, grid, kv, cu):
        assert nt == tiles(kind, causal, group, new[b], kv[b], blk) and 0 <= tile and cnt >= 1 and tile + cnt <= nt
        assert 0 <= c0 <= cta <= c1 < grid
        parts.setdefault((b, h, blk), []).append((cta, tile, cnt, c0, c1))
    want = 0
    for b, (n, t) in enumerate(zip(new, kv)):
        blk = 0
        while (nt := tiles(kind, causal, group, n, t, blk)) is not None:
            for h in range(heads):
                got = parts[b, h, blk]
                assert [x[0] for x in got] == list(range(got[0][3], got[0][4] + 1))  # the owners that each part names
                at = 0
                for _, tile, cnt, *own in got:
                    assert tile == at and own == [got[0][3], got[0][4]]
                    at += cnt
                assert at == nt
                want += 1
            blk += 1
    assert want == len(parts)


@pytest.mark.parametrize("kind", ["rows8", "rows16", "chunk"])
@pytest.mark.parametrize("seed", range(20))
def test_a_walk_ends_whatever_the_lengths_turn_into(cut, kind, seed):
    """Lengths and offsets that change between two reads of a call (a caller's mistake) must not make it loop, nor reach past
    the sequences: the loops that look for a share's beginning and for the next sequence end with the batch."""
    rng = random.Random(100 + seed)
    batch, heads, group, grid = rng.choice([1, 3, 33, 70]), rng.choice([1, 4]), rng.choice([1, 4]), 24
    new = [rng.choice([1, 1, 5, 200]) for _ in range(batch)]
    kv = [n + rng.randint(0, 9000) for n in new]
    cu = [sum(new[:i]) for i in range(batch + 1)]
    changes = []
    when = rng.randint(1, 40)
    if seed % 2:  # all of them short, or no new tokens at all
        changes = [(when, 0, i, rng.choice([0, 1])) for i in range(batch)] + [(when, 1, i, 0) for i in range(batch + 1) if seed % 4 == 1]
    else:
        changes = [(rng.randint(1, 60), rng.randint(0, 1), rng.randrange(batch), rng.choice([0, 3, 1 << 30, -9])) for _ in range(9)]
    for cta, b, h, blk, tile, cnt, nt, c0, c1 in cut(kind, rng.randint(0, 1), group, heads, grid, kv, cu, changes=changes):
        assert 0 <= b < batch and 0 <= h < heads and blk >= 0 and tile >= 0 and cnt >= 1 and tile + cnt <= nt
        assert 0 <= c0 < grid and 0 <= c1 < grid
