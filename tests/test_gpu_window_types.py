"""GPU: layers of another type than the plan's are refused behind a window as without one."""

import pytest
import torch

from gpu_helpers import workspace
from mstar_amd.paged_attention import PagedDecodeWrapper, PagedPrefillWrapper

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("window", [{}, {"window_left": 3}])
@pytest.mark.parametrize("new", [[1, 1], [40, 1], [40, 60]])
def test_fp32_layer_under_a_bf16_plan(gpu, new, window):
    index = [torch.tensor(x, dtype=torch.int32) for x in ([0, 4, 8], list(range(8)), [5, 9])]
    layer = torch.zeros(8, 2, 16, 2, 128, device=gpu)
    q = torch.zeros(sum(new), 8, 128, dtype=torch.bfloat16, device=gpu)
    f = PagedPrefillWrapper(workspace(gpu, 64 << 20), 8, 2, 128, 16, device=gpu)
    f.plan(torch.tensor([0, new[0], sum(new)], dtype=torch.int32), *index)
    with pytest.raises(RuntimeError):
        f.run(q, layer, **window)
    if max(new) == 1:
        w = PagedDecodeWrapper(workspace(gpu, 64 << 20), 8, 2, 128, 16, device=gpu)
        w.plan(*index)
        with pytest.raises(RuntimeError):
            w.run(q, layer, **window)
