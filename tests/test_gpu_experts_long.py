"""GPU checks of plans of many slots, whose runs' counts are added up by a launch of their own."""
import numpy as np
import pytest
import torch

import mx_format as mx
from test_gpu_mxfp4 import say

pytestmark = pytest.mark.gpu

RUN = 4096                                                   # slots of a run


@pytest.mark.parametrize("dtype", [torch.int32, torch.int64])
@pytest.mark.parametrize("R,E", [(64 * RUN, 7), (64 * RUN + 1, 7), (65 * RUN, 130), (65 * RUN + 1, 1024), (81 * RUN - 3, 1),
                                 (3_000_001, 65), (20_000_000, 64)])
def test_long_plan(backend, gpu, R, E, dtype):
    say("long plan", R, E, dtype)
    ids = np.random.RandomState(E).randint(-1, E + 1, R)     # -1 and E: unused
    ids[R // 3:R // 2] = E // 2                              # a run of one expert's alone
    t = torch.from_numpy(ids).to(dtype).cuda()
    k = next(k for k in (3, 2, 1) if R % k == 0)
    plan = backend.sort_tokens_by_expert(t.view(-1, k), E)
    for got, want in zip(plan, mx.plan(ids.reshape(-1, k), E)):
        assert np.array_equal(got.cpu().numpy(), want)


def test_long_plan_in_a_graph(backend, gpu):
    """Captured and replayed with other choices each time."""
    R, E = 70 * RUN, 40
    g = torch.Generator(device="cuda").manual_seed(1)
    ids = torch.randint(-1, E, (R, 1), generator=g, device="cuda")
    backend.sort_tokens_by_expert(ids, E)
    torch.cuda.synchronize()
    graph, held = torch.cuda.CUDAGraph(), ids.clone()
    with torch.cuda.graph(graph):
        plan = backend.sort_tokens_by_expert(held, E)
    for i in range(4):
        new = torch.randint(-1, E, (R, 1), generator=g, device="cuda")
        held.copy_(new)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(plan, backend.sort_tokens_by_expert(new, E)))
