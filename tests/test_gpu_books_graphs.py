"""GPU test of two captured services of a pool's books, with everything that the graphs read and write kept alive by the test."""
import pytest
import torch

from test_gpu_books import BF, E4, I32, _books

pytestmark = pytest.mark.gpu


def test_two_kept_graphs(dev):
    # replayed in turn and together, with other allocations in between: nothing is shared between them
    import tabicl_mi355_paged as paged
    runs = []
    for seed in (1, 2):
        table, n, free, fc, _ = _books(dev, seed, [40, 200, 0], 30, 16, spare=60)
        P = free.numel()
        g = torch.Generator(device=dev).manual_seed(seed)
        kp, vp = (torch.randn(P, 8, 16, 64, generator=g, device=dev).to(E4) for _ in range(2))
        held = (table, n, free, fc, kp, vp, torch.ones(P, 8, 2, device=dev), torch.randn(3, 8, 1, 64, generator=g, device=dev).to(BF),
                torch.tensor([3, 1, 9], dtype=I32, device=dev), torch.zeros(P, 8, 2, 64, dtype=torch.int8, device=dev),
                torch.zeros(P, 8, device=dev))

        def step(table, n, free, fc, kp, vp, scales, q, count, bnd, bs):
            granted = paged.paged_reserve(table, n, count, free, fc, 16)
            paged.paged_bounds(kp, table, n, bnd, bs, None, None, scales)
            index = paged.paged_select(q, bnd, bs, table, n, 16, 4)
            outs = granted, index, paged.paged_sparse_attention(q, kp, vp, table, n, index, scales=scales), \
                paged.paged_attention(q, kp, vp, table, n, scales=scales)
            paged.paged_release(table, n, free, fc, 16)
            return outs

        want = [t.clone() for t in step(*held)]
        stream, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            got = step(*held)
        runs.append((graph, got, want, stream, held))
    torch.cuda.synchronize()
    for together in (False, True, True, False, True):
        for _, got, _, _, _ in runs:
            for t in got:
                t.view(torch.uint8).fill_(7)
        other = [torch.full((k,), -1, dtype=I32, device=dev) for k in (3, 4, 60, 90, 5000, 100000)]
        torch.cuda.synchronize()
        for graph, _, _, stream, _ in runs:
            with torch.cuda.stream(stream if together else torch.cuda.current_stream()):
                graph.replay()
        torch.cuda.synchronize()
        assert all((t == -1).all() for t in other)
        for _, got, want, _, _ in runs:
            for a, b in zip(got, want):
                assert torch.equal(a, b)
