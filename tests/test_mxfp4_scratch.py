"""
Products over microscaled 4-bit weights that need scratch (a few bfloat16 rows over a large matrix, which go in pieces): captured and replayed,
on two streams at once, and which weights take them.
"""

from __future__ import annotations

import pytest
import torch

import mxfp4_plain as plain
from test_mxfp4 import DEV, check, f64, held, numbers, sums_bound
from tinyserve_llm_b200.ops import MXFP4

N, K = 2600, 2176            # 5.7 M numbers
ROWS = (9, 16, 12)


@pytest.fixture(scope="module")
def ops():
    from tinyserve_llm_b200.ops import get_ops
    return get_ops()


@pytest.fixture(scope="module")
def weight():
    w = f64(numbers((N, K), torch.float32, 31, 0.02))
    return w, held(w, DEV)


def shifted(q: MXFP4, offset: int, ld: int) -> MXFP4:
    """The same matrix with its rows of codes `ld` bytes apart, the first one `offset` bytes behind a 512-byte boundary."""
    room = torch.zeros((q.rows * ld + offset,), dtype=torch.uint8, device=DEV)
    codes = room.as_strided((q.rows, q.codes.shape[1]), (ld, 1), offset)
    codes.copy_(q.codes)
    return MXFP4(codes, q.scales, q.cols)


@pytest.mark.gpu
def test_weights_that_do_not_take_pieces(ops, weight):
    """Rows of codes that start 16 bytes off a 32-byte boundary: right, without the pieces' launch; aligned ones have it, and count it."""
    w, q = weight
    x = numbers((9, K), torch.bfloat16, 32).to(DEV)
    values = plain.rounded(w)
    want, off = f64(x) @ values.T, sums_bound(f64(x), values, K)
    line = q.codes.shape[1]
    for offset, ld, launches in ((0, line, 2), (16, line, 1), (0, line + 16, 1), (32, line + 32, 2)):
        moved = shifted(q, offset, ld)
        before = ops.launches
        y = ops.linear_mxfp4(x, moved, out_dtype=torch.float32)
        assert ops.launches - before == launches, (offset, ld)
        check(y, want, off)
    torch.cuda.synchronize()
    ops.check_device_errors()


@pytest.mark.gpu
def test_scratch_in_a_graph(ops, weight):
    """Captured once, replayed on new rows, beside eager calls between the replays."""
    _, q = weight
    xs = [numbers((m, K), torch.bfloat16, m).to(DEV) for m in ROWS]

    def both(x):
        return ops.linear_mxfp4(x, q), ops.linear_gated_mxfp4(x, q, "silu")

    for x in xs:
        both(x)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    before = ops.launches
    with torch.cuda.graph(graph):
        got = [both(x) for x in xs]
    assert ops.launches - before == 4 * len(xs)
    for seed in (40, 50):
        for i, x in enumerate(xs):
            x.copy_(numbers((ROWS[i], K), torch.bfloat16, seed + i).to(DEV))
        graph.replay()
        eager = [both(x) for x in xs]
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for one, other in zip(got, eager) for a, b in zip(one, other))
    ops.check_device_errors()


@pytest.mark.gpu
def test_two_graphs_that_share_a_pool(ops, weight):
    """Two captured graphs over one memory pool, replayed one behind the other: each gives its own rows' product."""
    _, q = weight
    xs = [numbers((m, K), torch.bfloat16, 60 + m).to(DEV) for m in ROWS[:2]]
    alone = [ops.linear_mxfp4(x, q).clone() for x in xs]
    torch.cuda.synchronize()
    graphs, got = [torch.cuda.CUDAGraph() for _ in xs], []
    for i, x in enumerate(xs):
        with torch.cuda.graph(graphs[i], pool=graphs[0].pool() if i else None):
            got.append(ops.linear_mxfp4(x, q))
    for _ in range(3):
        for i, graph in enumerate(graphs):
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(got[i], alone[i])
    ops.check_device_errors()


@pytest.mark.gpu
def test_scratch_on_two_streams(ops, weight):
    _, q = weight
    xs = [numbers((m, K), torch.bfloat16, 70 + m).to(DEV) for m in ROWS[:2]]
    alone = [ops.linear_mxfp4(x, q) for x in xs]
    torch.cuda.synchronize()
    streams, found = [torch.cuda.Stream() for _ in xs], [[], []]
    for _ in range(30):
        for i, (stream, x) in enumerate(zip(streams, xs)):
            with torch.cuda.stream(stream):
                found[i].append(ops.linear_mxfp4(x, q))
    torch.cuda.synchronize()
    for a, results in zip(alone, found):
        assert all(torch.equal(a, r) for r in results)
    ops.check_device_errors()


def test_what_is_no_matrix_in_four_bits_is_refused():
    """A bfloat16 weight, or one's codes alone, where an MXFP4 is wanted; a class derived from it is one."""
    from tinyserve_llm_b200.ops import KernelError, Ops
    ops, x = Ops.__new__(Ops), torch.zeros((4, 64), dtype=torch.bfloat16)
    for call in (lambda w: ops.linear_mxfp4(x, w), lambda w: ops.linear_gated_mxfp4(x, w, "silu"), ops.dequantize_mxfp4):
        for bad in (x, None, torch.zeros((4, 32), dtype=torch.uint8)):
            with pytest.raises(KernelError, match="MXFP4"):
                call(bad)

    class Derived(MXFP4):
        pass

    q = Derived(torch.zeros((4, 32), dtype=torch.uint8), torch.zeros((4, 16), dtype=torch.uint8)[:, :2], 64)
    other = MXFP4(torch.zeros((4, 16), dtype=torch.uint8), torch.zeros((4, 16), dtype=torch.uint8)[:, :1], 32)
    with pytest.raises(KernelError, match=r"x is \(4, 64\), the weight has rows of 32"):
        ops.linear_mxfp4(q, other)
