"""What the grouped products, label log probabilities and the AdamW step refuse, on any machine."""
import ctypes

import pytest
import torch

from image_classification_amd import _lib, ops


def z(*shape, **kw):
    return torch.zeros(*shape, **kw)


I32 = dict(dtype=torch.int32)
I64 = dict(dtype=torch.int64)


@pytest.mark.parametrize("call", [
    lambda: ops.group_rows(z(4, **I64), 3),
    lambda: ops.group_rows(z(4, 2, **I32), 3),
    lambda: ops.group_rows(z(4, **I32), 0),
    lambda: ops.group_rows(z(4, **I32), (1 << 26) + 1),
    lambda: ops.group_rows(z(4, **I32), 3),                                    # not on a GPU
    lambda: ops.grouped_matmul(z(4, 8), z(2, 3, 9), z(3, **I64)),              # widths
    lambda: ops.grouped_matmul(z(4, 8), z(3, 8), z(3, **I64)),                 # w not 3-D
    lambda: ops.grouped_matmul(z(4, 8), z(2, 8, 3).transpose(1, 2), z(3, **I64)),
    lambda: ops.grouped_matmul(z(4, 8), z(0, 3, 8), z(1, **I64)),
    lambda: ops.grouped_matmul(z(4), z(2, 3, 8), z(3, **I64)),
    lambda: ops.grouped_matmul(z(8, 4).t(), z(2, 3, 8), z(3, **I64)),          # columns adjacent, not rows
    lambda: ops.grouped_matmul(z(1, 8).expand(4, 8), z(2, 3, 8), z(3, **I64)),  # rows overlap
    lambda: ops.grouped_matmul(z(4, 8), z(2, 3, 8, dtype=torch.float16), z(3, **I64)),
    lambda: ops.grouped_matmul(z(4, 8, dtype=torch.float64), z(2, 3, 8, dtype=torch.float64), z(3, **I64)),
    lambda: ops.grouped_matmul(z(4, 8), z(2, 3, 8), z(3, **I64)),              # not on a GPU
    lambda: ops.grouped_matmul_dx(z(4, 8), z(2, 3, 8), z(3, **I64)),           # dy has `out` columns
    lambda: ops.grouped_matmul_dw(z(4, 3), z(5, 8), z(3, **I64)),
    lambda: ops.grouped_matmul_dw(z(4, 3), z(4, 8, dtype=torch.float16), z(3, **I64)),
    lambda: ops.grouped_matmul_dw(z(4, 0), z(4, 8), z(3, **I64)),
    lambda: ops.label_logprobs(z(4)),
    lambda: ops.label_logprobs(z(4, 0)),
    lambda: ops.label_logprobs(z(4, 5, dtype=torch.float64)),
    lambda: ops.label_logprobs(z(4, 5), top=6),
    lambda: ops.label_logprobs(z(4, 50), top=33),
    lambda: ops.label_logprobs(z(4, 5), top=-1),
    lambda: ops.label_logprobs(z(4, 5), temperature=0.0),
    lambda: ops.label_logprobs(z(4, 5), temperature=float("inf")),
    lambda: ops.label_logprobs(z(4, 5), temperature=float("nan")),
    lambda: ops.label_logprobs(z(4, 5)),                                       # not on a GPU
    lambda: ops.label_logprobs_grad(z(4, 5), None, z(4), z(4), z(4)),
    lambda: ops.label_logprobs_grad(z(4, 5), z(4, **I64), None, z(4), z(4)),
    lambda: ops.adamw_states([z(3)], 16),
    lambda: ops.adamw_step([z(3)], [], z(256), z(256), lr=1e-3, step=1),
    lambda: ops.adamw_step([z(3)], [z(3)], z(256), z(256), lr=1e-3, step=1, scales=z(2, 1)),
    lambda: ops.adamw_step([z(3)], [z(3)], z(256, dtype=torch.float16), z(256), lr=1e-3, step=1),
    lambda: ops.adamw_step([z(3)], [z(3)], z(256), z(256), lr=1e-3, step=1),   # not on a GPU
    lambda: ops.adamw_state_values(z(300, dtype=torch.uint8), z(300, dtype=torch.uint8), z(2, 1)),
    lambda: ops.adamw_state_values(z(256, dtype=torch.uint8), z(256, dtype=torch.uint8), z(1, 1)),
    lambda: ops.adamw_state_values(z(256, dtype=torch.uint8), z(256, dtype=torch.uint8), z(2, 1)),
])
def test_refused_before_anything_is_launched(call):
    with pytest.raises(ValueError):
        call()


def test_a_handle_is_asked_for():
    lib = _lib.load()
    for name, args in (("ic_group_rows", 9), ("ic_grouped_matmul", 15), ("ic_grouped_matmul_dx", 15),
                       ("ic_grouped_matmul_dw", 17), ("ic_label_logprobs", 18),
                       ("ic_label_logprobs_grad", 16), ("ic_adamw_step", 18), ("ic_adamw_state_values", 8)):
        fn = getattr(lib, name)
        assert len(fn.argtypes) == args
        zeros = [None if t is ctypes.c_void_p else 0 for t in fn.argtypes]
        assert fn(*zeros) == 10003, name
        assert "invalid handle" in _lib.last_error()


def test_scratch_sizes():
    lib = _lib.load()
    assert lib.ic_group_rows_scratch(4096, 1000) == 0
    assert lib.ic_group_rows_scratch(1_000_000, 10_000) >= 12_000_000   # pairs and sorted codes
    # two partial tiles a workgroup: at most 256 x 2 x 256 x 256 floats, little for little work
    for t in (0, 1, 2):
        assert lib.ic_grouped_matmul_dw_scratch(0, 1, 8, 8, t) == 0          # nothing is cut
        assert lib.ic_grouped_matmul_dw_scratch(100, 50, 800, 80, t) == 0
        for n, e, k, out in ((1_000_000, 10_000, 128, 64), (65536, 16, 2048, 2048), (3_000_000, 1, 2048, 16),
                             (4097, 3, 8, 8)):
            assert 0 < lib.ic_grouped_matmul_dw_scratch(n, e, k, out, t) <= 2 * 256 * 256 * 256 * 4
    assert lib.ic_label_logprobs_scratch(100_000, 1000, 1, 5) == 0
    assert lib.ic_label_logprobs_scratch(4, 65536, 0, 5) > 0
    assert lib.ic_label_logprobs_scratch(4, 65536, 9, 5) == 0


# -- host arithmetic of the tile numbering (what find_group and the grids rely on) ---------------------------
def test_every_tile_of_ragged_groups_has_a_number():
    import numpy as np
    rng = np.random.default_rng(0)
    for trial in range(300):
        groups = int(rng.integers(1, 12))
        bm = int(rng.choice([16, 64, 128, 512]))
        sizes = rng.choice([0, 0, 1, bm - 1, bm, bm + 1, 3 * bm, int(rng.integers(0, 5 * bm))], groups)
        off = np.concatenate([[0], np.cumsum(sizes)])
        n = int(off[-1] + rng.integers(0, 3 * bm))
        first = np.array([off[e] // bm + e for e in range(groups + 1)])
        total = n // bm + groups + 1
        assert (np.diff(first) >= 1).all()
        ends = np.append(off[1:], n)
        for e in range(groups + 1):
            tiles = -(-(ends[e] - off[e]) // bm)
            nxt = first[e + 1] if e < groups else total
            assert first[e] + tiles <= nxt


@pytest.mark.parametrize("seed", range(40))
def test_the_line_of_a_weight_gradient_is_covered_once(seed):
    # the units of every tile of every group: each stage in exactly one workgroup's run, pieces of a
    # cut tile in at most one begin and one end place of a workgroup, every tile joined exactly once
    import numpy as np
    rng = np.random.default_rng(seed)
    kk = int(rng.choice([32, 64]))
    groups, tiles, wgs = int(rng.integers(1, 9)), int(rng.integers(1, 5)), int(rng.integers(1, 40))
    sizes = rng.choice([0, 1, kk, kk + 1, int(rng.integers(0, 2000))], groups)
    off = np.concatenate([[0], np.cumsum(sizes)])
    first = [int(off[e]) // kk + e for e in range(groups + 1)]
    line = first[groups] * tiles

    def place(u):
        e = max(e for e in range(groups + 1) if first[e] <= u // tiles)
        stages = int(off[e + 1]) // kk + 1 - int(off[e]) // kk
        inside = u - first[e] * tiles
        assert e < groups and 0 <= inside // stages < tiles
        return e, inside // stages, inside % stages, stages

    seen, pieces, whole, joined = {}, {}, set(), set()
    for w in range(wgs):
        u, u1 = line * w // wgs, line * (w + 1) // wgs
        while u < u1:
            e, t, st, stages = place(u)
            run = min(stages - st, u1 - u)
            assert stages * kk >= sizes[e]
            for i in range(st, st + run):
                assert (e, t, i) not in seen
                seen[e, t, i] = w
            if st == 0 and run == stages:
                whole.add((e, t))
            else:
                key = (w, 1 if st == 0 else 0)
                assert key not in pieces
                pieces[key] = (e, t)
            u += run
    assert len(seen) == line
    for w in range(wgs - 1):
        u0, u1 = line * w // wgs, line * (w + 1) // wgs
        if u1 >= line or u0 >= u1:
            continue
        e, t, st, stages = place(u1)
        begin, end = u1 - st, u1 - st + stages
        if st == 0 or begin < u0:
            continue
        mine = []
        for v in range(w, wgs):
            if v > w and line * v // wgs >= end:
                break
            if v > w and line * v // wgs == line * (v + 1) // wgs:
                continue
            mine.append((v, 1 if v == w else 0))
        assert [pieces.pop(key) for key in mine] == [(e, t)] * len(mine)
        assert (e, t) not in joined
        joined.add((e, t))
    assert not pieces and not (whole & joined)
    assert whole | joined == {(e, t) for e in range(groups) for t in range(tiles)}


@pytest.mark.parametrize("seed", range(40))
def test_the_ends_inside_a_cut_tile_share_its_join(seed):
    # the join's workgroups: every element of a cut tile is taken by exactly one of the ends that lie
    # inside the tile, whatever the runs (empty ones among them), and all agree on the tile's workgroups
    import numpy as np
    rng = np.random.default_rng(100 + seed)
    kk = int(rng.choice([32, 64]))
    groups, tiles, wgs = int(rng.integers(1, 6)), int(rng.integers(1, 4)), int(rng.integers(2, 60))
    each, chunks = int(rng.choice([1, 4, 16])), 16
    sizes = rng.choice([0, 1, kk, kk + 1, int(rng.integers(0, 4000))], groups)
    off = [int(o) for o in np.concatenate([[0], np.cumsum(sizes)])]
    first = [off[e] // kk + e for e in range(groups + 1)]
    line = first[groups] * tiles
    run_of = {}
    for w in range(wgs):
        for u in range(line * w // wgs, line * (w + 1) // wgs):
            run_of[u] = w
    begins, u = {}, 0
    for e in range(groups):
        stages = off[e + 1] // kk + 1 - off[e] // kk
        for _ in range(tiles):
            for q in range(u, u + stages):
                begins[q] = (u, u + stages)
            u += stages
    assert u == line
    taken = {}
    for w in range(wgs - 1):
        u1 = line * (w + 1) // wgs
        if u1 >= line or begins[u1][0] == u1:
            continue
        begin, end = begins[u1]
        lo, hi = ((begin + 1) * wgs - 1) // line, (end * wgs - 1) // line
        assert lo == run_of[begin] and hi == run_of[end - 1] and lo <= w < hi
        for x in range(each):
            mine = (w - lo) * each + x
            assert 0 <= mine < (hi - lo) * each
            for at in range(mine, chunks, (hi - lo) * each):
                assert (begin, at) not in taken
                taken[begin, at] = w
    cut = {b for b, end in begins.values() if run_of[b] != run_of[end - 1]}
    assert set(taken) == {(b, at) for b in cut for at in range(chunks)}


def test_memory_that_is_shared():
    wide = z(6, 40)
    apart = [(wide[:, :8], wide[:, 8:20]), (wide[:, 30:], wide[:, :30]), (wide[:3], wide[3:]),
             (z(4, 8), z(4, 8)), (wide[0:1, :8], wide[0:1, 8:]), (z(0, 8), z(0, 8))]
    for a, b in apart:
        ops._check_apart(a, b)
        ops._check_apart(b, a)
    shared = [(wide, wide), (wide[:, :8], wide[:, 7:20]), (wide[:4], wide[3:]), (wide[:, 4:12], wide),
              (z(30).as_strided((4, 3), (6, 1)), None)]
    flat = shared.pop()[0]
    shared.append((flat, flat.as_strided((3, 3), (7, 1))))      # other row strides: refused unless apart
    for a, b in shared:
        with pytest.raises(ValueError, match="share no memory"):
            ops._check_apart(a, b)
        with pytest.raises(ValueError, match="share no memory"):
            ops._check_apart(b, a)


@pytest.mark.parametrize("seed", range(20))
def test_whole_tiles_of_a_weight_gradient_are_dealt_once(seed):
    # few rows: runs that begin and end with tiles (the unit a run begins with, worked out from its tile)
    import numpy as np
    rng = np.random.default_rng(200 + seed)
    kk = int(rng.choice([32, 64]))
    groups, tiles = int(rng.integers(1, 9)), int(rng.integers(1, 6))
    wgs = int(rng.integers(1, groups * tiles + 1))
    sizes = rng.choice([0, 0, 1, kk, int(rng.integers(0, 4 * kk))], groups)
    off = [int(o) for o in np.concatenate([[0], np.cumsum(sizes)])]
    line = (off[groups] // kk + groups) * tiles

    def begin(w):
        t = groups * tiles * w // wgs
        e = t // tiles
        if e >= groups:
            return line
        stages = off[e + 1] // kk + 1 - off[e] // kk
        return (off[e] // kk + e) * tiles + t % tiles * stages

    assert begin(0) == 0 and begin(wgs) == line
    starts, u = set(), 0
    for e in range(groups):
        for _ in range(tiles):
            starts.add(u)
            u += off[e + 1] // kk + 1 - off[e] // kk
    assert u == line
    at = [begin(w) for w in range(wgs + 1)]
    assert at == sorted(at) and set(at[:-1]) <= starts and len(set(at)) == wgs + 1
