"""The paged full-attention layer as a module's replacement."""

from __future__ import annotations

import pytest
import torch

from test_gpu_paged import BF, _ints

pytestmark = pytest.mark.gpu


def test_paged_layer_keeps_no_graph(device):
    from lightreason_amd.attention import AttentionDecode
    from lightreason_amd.paged import PageTable, paged_layer

    def weight(*shape):
        return torch.nn.Parameter(0.02 * torch.randn(*shape, dtype=BF, device=device))
    attn = AttentionDecode(q_proj=weight(8192, 2048), k_proj=weight(512, 2048), v_proj=weight(512, 2048),
                           o_proj=weight(2048, 4096), q_norm=weight(256), k_norm=weight(256))
    pt = PageTable(2, 10, 16, device=device)
    kc, vc = pt.new_cache(1)
    plan = pt.plan(_ints([3, 1], device), 4)
    hidden = torch.randn(4, 2048, dtype=BF, device=device, requires_grad=True)
    cos = torch.ones(16, 64, dtype=BF, device=device)
    out = paged_layer(attn, hidden, cos, cos, kc[0], vc[0], pt, plan)
    assert not out.requires_grad and out.grad_fn is None
    with torch.no_grad():
        assert torch.equal(out, paged_layer(attn, hidden, cos, cos, kc[0], vc[0], pt, plan))
