"""The workspace of a product with a tensor is that of the operand's own device: the library's rule goes by its SM
count."""
import contextlib
import types

import torch

from custom_matmul_kernels_b200 import mx


def test_asked_on_the_operands_device(monkeypatch):
    current, asked = [0], []

    @contextlib.contextmanager
    def device(index):
        before, current[0] = current[0], index
        yield
        current[0] = before

    def query(l, m, n, k, layout):
        asked.append(current[0])
        return 1000 * current[0] + m

    monkeypatch.setattr(torch.cuda, "device", device)
    monkeypatch.setattr(mx, "load_library", lambda: types.SimpleNamespace(fbmm_mx4_bmm_tensor_workspace_bytes=query))
    mx._product_workspace.cache_clear()
    try:
        for _ in range(2):  # from whichever device is current, and from the cache
            for index in (0, 3, 1):
                assert mx._product_workspace(index, 1, 7, 64, 64, ord("n")) == 1000 * index + 7
        assert asked == [0, 3, 1] and current == [0]
    finally:
        mx._product_workspace.cache_clear()
