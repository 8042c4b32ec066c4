"""CPU tests of the hidden-state operators' planner: the launches of a call, as
its C entry point makes them, over buffers that nothing reads (head_launches.py)."""
from __future__ import annotations

import random

import pytest

import head_launches as HL
import head_shapes as SH


# rows, hidden, vocabulary whose last piece is split into more parts than the
# first when each piece's parts are derived from its own length
PARTS = [("bf16", 1529, 256, 248320), ("f32", 1472, 256, 151936), ("f32", 614, 512, 129280),
         ("f32", 186, 3094, 200899), ("bf16", 404, 580, 221326), ("f32", 1466, 256, 151936),
         ("f16", 686, 472, 110778), ("bf16", 411, 240, 205007)]


@pytest.mark.parametrize("case", PARTS, ids=lambda c: "-".join(map(str, c)))
def test_parts_of_later_pieces(case):
    """d_x's float32 parts are written, added to and joined piece after piece."""
    for want_weight in (True, False):
        need, launches = HL.head_loss_backward(*case, want_weight=want_weight)
        dx = [l for l in launches if l.kind == HL.PARTIAL and l.roles == HL.ROLES.index("NN")]
        assert len(dx) > 1 and dx[0].parts > 1, "the case is no longer one of split pieces"
        HL.check_workspace(need, launches)


@pytest.mark.parametrize("m,n", [(1, (1 << 21) + 1), (40, 3000001), (700, 1 << 22)])
@pytest.mark.parametrize("bias", [False, True])
def test_products_follow_the_pass_that_writes_what_they_read(m, n, bias):
    """The gradient at the pre-activations is written by the pass over d_out and
    read where it lies, however long its rows are."""
    for dtype in HL.DTYPES:
        need, launches = HL.linear_backward(dtype, m, 64, n, activation=2, bias=bias)
        HL.check_workspace(need, launches)
        dz = next(l.out for l in launches if l.kind == HL.COL_SUM)
        read = [l.a for l in launches if l.kind in (HL.STORE, HL.PARTIAL)]
        assert len(read) == 2 and all(p == dz for p in read)


def test_sums_of_many_rows_are_joined_by_more_waves():
    """The size of test_head_bias_gradient_sums_in_float32 with the most rows."""
    need, launches = HL.head_loss_backward("bf16", 20011, 72, 333, bias=True)
    HL.check_workspace(need, launches)
    assert [l.chunks for l in launches if l.kind == HL.COL_SUM_JOIN][0] > 256


def _log_int(rng, low, high):
    return int(round(low * (high / low) ** rng.random()))


def test_workspace_of_any_size():
    """Every call's launches stay inside its workspace, over sizes, types and
    layouts drawn at random."""
    rng = random.Random(20)
    for i in range(4000):
        dtype, layout = rng.choice(list(HL.DTYPES)), rng.choice(["dense", "pad", "odd"])
        m, k = _log_int(rng, 1, 4096), _log_int(rng, 1, 8192)
        v = rng.choice([32000, 128256, 151936, _log_int(rng, 1, 262144)])
        n = _log_int(rng, 1, 16384)
        kw = dict(bias=rng.random() < 0.5, want_x=rng.random() < 0.8)
        kw["want_weight"] = rng.random() < 0.8 or not (kw["bias"] or kw["want_x"])
        act = rng.randrange(3)
        for f, args, more in ((HL.linear, (m, k, n), {}),
                              (HL.linear_backward, (m, k, n), dict(kw, activation=act)),
                              (HL.head_loss, (m, k, v), {}),
                              (HL.head_loss_backward, (m, k, v), kw)):
            need, launches = f(dtype, *args, layout, **more)
            try:
                HL.check_workspace(need, launches)
            except AssertionError as e:
                raise AssertionError(f"{f.__name__} {dtype} {args} {layout} {more}: {e}") from None


# every product of an operator (operator, launch, roles of the operands) and the
# shapes that SHAPES has to reach for it.  "parts": a reduction split over work-groups.
ALL = "256 128 64 128x2 64x4 loose128 loose64 loose64x4"
F32 = ALL[4:]
TAKEN = {
    ("head", "16", "gradient", "NT"): "256 128 64 128x2 64x4 loose128",
    ("head", "16", "parts", "NN"): "128 64 64x4 loose128 loose64 loose64x4",
    ("head", "16", "parts", "TN"): "128 64 64x4",
    ("head", "16", "statistics", "NT"): "256 128 64 128x2 64x4 loose128",
    ("head", "16", "store", "NN"): "256 128 64 128x2 64x4 loose64",
    ("head", "16", "store", "TN"): ALL,
    ("head", "f32", "gradient", "NT"): "128 64 128x2 64x4 loose128",
    ("head", "f32", "parts", "NN"): "128 64 128x2 64x4 loose128 loose64x4",
    ("head", "f32", "parts", "TN"): "128 64 128x2 64x4 loose64x4",
    ("head", "f32", "statistics", "NT"): "128 64 128x2 64x4 loose128",
    ("head", "f32", "store", "NN"): "128 64 128x2 64x4 loose128 loose64",
    ("head", "f32", "store", "TN"): "128 64 128x2 loose128 loose64 loose64x4",
    ("linear", "16", "out", "NT"): "256 128 64 128x2 loose128 loose64",
    ("linear", "16", "parts", "NT"): "64 64x4 loose64 loose64x4",
    ("linear", "f32", "out", "NT"): "128 64 128x2 loose128 loose64",
    ("linear", "f32", "parts", "NT"): "128 128x2 64x4 loose128 loose64x4",
    ("linear_backward", "16", "parts", "NN"): "128 64 64x4 loose128 loose64 loose64x4",
    ("linear_backward", "16", "parts", "TN"): "128 64 64x4 loose128 loose64 loose64x4",
    ("linear_backward", "16", "store", "NN"): "256 128 64 128x2 64x4 loose128 loose64",
    ("linear_backward", "16", "store", "TN"): "256 128 64 128x2 loose128 loose64 loose64x4",
    ("linear_backward", "f32", "parts", "NN"): "128 64 128x2 64x4 loose128 loose64x4",
    ("linear_backward", "f32", "parts", "TN"): "128 64 128x2 64x4 loose128 loose64x4",
    ("linear_backward", "f32", "store", "NN"): "128 64 128x2 loose128 loose64",
    ("linear_backward", "f32", "store", "TN"): "128 64 128x2 64x4 loose128 loose64",
}


def _products(op, dtype, m, k, n, layout):
    """The products of a case: (operator, dtype, launch, roles), shape and launch."""
    kinds = {HL.LINEAR: "out", HL.STATS: "statistics", HL.GRAD: "gradient", HL.STORE: "store",
             HL.PARTIAL: "parts"}
    calls = {"linear": [(HL.linear, {})], "linear_backward": [(HL.linear_backward, {"activation": 2})],
             "head": [(HL.head_loss, {}), (HL.head_loss_backward, {"bias": True})]}[op]
    for f, kw in calls:
        need, launches = f("bf16" if dtype == "16" else dtype, m, k, n, layout, **kw)
        HL.check_workspace(need, launches)
        for l in launches:
            if l.kind in kinds:
                yield (op, dtype, kinds[l.kind], HL.ROLES[l.roles]), HL.TILES[l.tile], l


def test_sizes_take_every_shape():
    """The sizes that the GPU tests run take every tile shape, so that a constant of
    the planner cannot change and leave one untested."""
    taken = {}
    for case in SH.SHAPES:
        for product, tile, _ in _products(*case):
            taken.setdefault(product, set()).add(tile)
    for product, tiles in TAKEN.items():
        assert set(tiles.split()) <= taken[product], (product, set(tiles.split()) - taken[product])


@pytest.mark.parametrize("slabs,case", list(enumerate(SH.LAST_PIECES, 1)), ids=str)
def test_last_pieces_of_a_few_slabs(slabs, case):
    got = [(tile, l) for p, tile, l in _products("head", "16", *case, "dense") if p[2:] == ("parts", "NN")]
    assert len(got) > 1 and all(tile == "256" for tile, _ in got)
    assert got[-1][1].accumulate and got[-1][1].slabs == slabs


@pytest.mark.parametrize("case", SH.COPIED, ids=str)
def test_weights_copied_in_pieces(case):
    dtype, m, k, v, layout = case
    for f in (HL.head_loss, HL.head_loss_backward):
        need, launches = f("bf16" if dtype == "16" else dtype, m, k, v, layout)
        HL.check_workspace(need, launches)
        packs = [l for l in launches if l.kind == HL.PACK and l.a >= HL.AT["weight"]]
        pieces = [l for l in launches if l.kind in (HL.STATS, HL.GRAD)]
        assert len(packs) == len(pieces) == 3 and pieces[-1].n < pieces[0].n
        assert [p.m for p in packs] == [p.n for p in pieces]


@pytest.mark.parametrize("case", SH.STREAMED, ids=str)
def test_large_outputs_are_stored_past_the_caches(case):
    need, launches = HL.linear(*case, pre=True)
    out = [l for l in launches if l.kind == HL.LINEAR]
    assert len(out) == 1 and out[0].stream
    assert HL.TILES[out[0].tile] == ("128" if case[0] == "f32" else "256")
