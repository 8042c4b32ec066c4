"""CPU tests of the hidden-state operators' planner: the launches of a call, as
its C entry point makes them, over buffers that nothing reads (head_launches.py)."""
from __future__ import annotations

import random

import pytest

import head_launches as HL


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
