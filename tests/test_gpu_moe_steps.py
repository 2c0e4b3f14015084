"""GPU check of the mixture-of-experts layer step by step: each step against its definition in 64 bits on the step before
as the library made it, so that no 4-bit rounding of a neighbouring value comes between them."""
import importlib

import numpy as np
import pytest
import torch

import mx_format as mx
from conftest import PKG_NAME
from test_gpu_moe import layer
from test_gpu_mxfp4 import DTYPES, np64, rounded_once

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("T,k,E,D,F,G", [(1, 2, 4, 256, 512, 256), (9, 3, 5, 128, 96, 16), (40, 2, 3, 512, 256, None),
                                         (200, 2, 6, 320, 448, 64)])
def test_steps(backend, gpu, T, k, E, D, F, G, dtype):
    print("moe steps", T, k, E, D, F, G, dtype, flush=True)
    moe = layer(importlib.import_module(PKG_NAME + ".mxfp4_moe").Mxfp4MoE, E, D, F, G)
    g = torch.Generator().manual_seed(T)
    x, ids = torch.randn(T, D, generator=g).to(dtype).cuda(), torch.randint(-1, E, (T, k), generator=g).cuda()
    w = torch.rand(T, k, generator=g).cuda()
    out = moe(x, ids, w)

    plan = backend.sort_tokens_by_expert(ids, E)
    first = backend.mxfp4_expert_linear(x, moe.w1, moe.s1, plan, convrot_groupsize=G)
    h = torch.nn.functional.silu(first[:, :F]) * first[:, F:]
    rows = backend.mxfp4_expert_linear(h, moe.w2, moe.s2, plan, convrot_groupsize=G, sorted_rows=True)
    order, position, offsets = mx.plan(ids.cpu().numpy(), E)

    def product(a, wc, ws, got):
        """Experts' products of the quantizer's codes: K roundings of 2^-23 of the sum of magnitudes, then the output's."""
        a = mx.dequantize(*(t.cpu().numpy() for t in backend.quantize_mxfp4(a, G)))
        b = mx.dequantize(wc.cpu().numpy(), ws.cpu().numpy())
        for e in range(E):
            r = slice(offsets[e], offsets[e + 1])
            at = a[order[r] // k] if got is first else a[r]
            off = (a.shape[1] + 2) * 2.0 ** -23 * (np.abs(at) @ np.abs(b[e]).T)
            assert rounded_once(got[r], at @ b[e].T, off, dtype)

    product(x, moe.w1, moe.s1, first)
    product(h, moe.w2, moe.s2, rows)
    terms = np.where((position >= 0)[..., None], np64(rows)[np.maximum(position, 0)], 0) * np64(w)[..., None]
    assert rounded_once(out, terms.sum(axis=1), k * 2.0 ** -24 * np.abs(terms).sum(axis=1), dtype)
    assert moe(x.view(1, T, D), ids.view(1, T, k), w.view(1, T, k)).equal(out.view(1, T, D))
