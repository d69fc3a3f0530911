"""GPU: what the calls of a model share between row counts, streams and captured graphs."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def test_captured_rows_workspace_is_the_graphs_own():
    """The row-stationary assembly's scratch inside a captured graph belongs to that graph: not to
    the stream (whose buffer is replaced when a larger call comes), nor to another graph."""
    from computd_b200 import assembler

    d, r, k, rows = 64, 2, 8, 32
    g = torch.Generator(device="cuda").manual_seed(0)
    vectors = torch.randn((rows, 2 * d * r + d), device="cuda", generator=g).bfloat16()

    def inputs(M):
        return (torch.randn((M, d), device="cuda", generator=g).bfloat16(),
                torch.rand((M, k), device="cuda", generator=g),
                torch.randint(0, rows, (M, k), device="cuda", generator=g).int())

    def call(x):
        return assembler.lowrank_delta(*x, vectors, d, d, r, rows=True)

    seen = []
    make = assembler.lowrank_rows_workspace

    def noted(*a):
        ws = make(*a)
        seen.append(ws.data_ptr())
        return ws

    small, large, largest = inputs(40), inputs(400), inputs(4000)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graphs = []
    assembler.lowrank_rows_workspace = noted
    try:
        with torch.cuda.stream(side):
            want = [call(small).clone(), call(large).clone()]
            torch.cuda.synchronize()
            for x in (small, large):
                graph = torch.cuda.CUDAGraph()
                with torch.cuda.graph(graph, stream=side):
                    out = call(x)
                graphs.append((graph, out))
    finally:
        assembler.lowrank_rows_workspace = make
    eager, captured = seen[:2], seen[2:]
    assert not set(eager) & set(captured) and captured[0] != captured[1]
    with torch.cuda.stream(side):  # the stream's buffer is replaced, its memory goes to others
        call(largest)
        junk = [torch.full((1 << 20,), 255, dtype=torch.uint8, device="cuda") for _ in range(20)]
        for _ in range(5):
            for graph, _ in graphs:
                graph.replay()
    torch.cuda.synchronize()
    assert all(bool((x == 255).all()) for x in junk)
    for (_, out), x in zip(graphs, want):
        assert torch.equal(out, x)
