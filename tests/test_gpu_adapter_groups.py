"""Groups of rows that group_rows() did not make for these rows and adapters are refused before anything is launched."""
import pytest
import torch

import qgemm_amd as Q

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("native", [True, False])
def test_groups_of_another_size_are_refused(native, monkeypatch):
    if not native:
        monkeypatch.setattr(Q.ops, "_native_module", False)
    f = lambda *shape, dtype=torch.bfloat16: torch.zeros(*shape, dtype=dtype, device="cuda")  # noqa: E731
    y, x, A, B, u = f(4, 32), f(4, 64), f(2, 8, 64), f(2, 8, 32), f(4, 8, dtype=torch.float32)
    good = Q.group_rows(f(4, dtype=torch.int32), 2)
    n = good.words.numel()
    assert torch.equal(Q.add_adapters(y, x, A, B, Q.RowGroups(4, 2, good.words)), y)
    bad = [Q.RowGroups(4, 2, w) for w in (good.words[:n - 4], f(n + 4, dtype=torch.int32), f(2 * n, dtype=torch.int32)[::2], f(0, dtype=torch.int32), good.words.cpu())]
    bad += [Q.RowGroups(4, 2, Q.group_rows(f(200, dtype=torch.int32), 2).words), Q.RowGroups(4, 2, Q.group_rows(f(4, dtype=torch.int32), 3).words)]
    assert all(g.words.numel() != n or not g.words.is_contiguous() or not g.words.is_cuda for g in bad)
    for g in bad:
        for call in (lambda: Q.add_adapters(y, x, A, B, g), lambda: Q.add_adapters_backward(y, x, u, A, B, g)):
            with pytest.raises(ValueError):
                call()
    for w in (good.words.long(), good.words.float()):
        with pytest.raises(TypeError):
            Q.add_adapters(y, x, A, B, Q.RowGroups(4, 2, w))
    for rows, adapters in ((5, 2), (3, 2), (4, 3), (4, 1)):
        with pytest.raises((ValueError, Q.QgemmError)):
            Q.add_adapters(y, x, A, B, Q.RowGroups(rows, adapters, good.words))
