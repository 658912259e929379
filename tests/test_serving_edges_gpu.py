"""Serving operators on the GPU at the edges of what their documentation allows."""
import os
import subprocess
import sys

import pytest
import torch

pytestmark = pytest.mark.gpu

DEV = "cuda"
ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def _i(v):
    return torch.tensor(v, dtype=torch.int32, device=DEV)


def _decode_tables(B, P=16):
    """A step of ``B`` requests that each add a token, every third of them on a new page; checked by arithmetic."""
    from distrain_b200.ops import paged
    cached = [(P if i % 3 == 0 else 1 + i % (P - 1)) for i in range(B)]
    opens = [i for i in range(B) if i % 3 == 0]
    tables = torch.full((B, 2), -1, dtype=torch.int32, device=DEV)
    tables[:, 0] = torch.arange(B, dtype=torch.int32, device=DEV)
    free = torch.arange(B, B + len(opens), dtype=torch.int32, device=DEV)
    slots, pos = torch.full((B,), 99, dtype=torch.int32, device=DEV), torch.full((B,), 99, dtype=torch.int32, device=DEV)
    cu, total, used = _i([99] * (B + 1)), _i([99] * B), _i([99, 99])
    paged.page_tables(_i(cached), _i([1] * B), free, tables, slots, pos, cu, total, used, page_size=P)
    assert used.tolist() == [len(opens), 0] and cu.tolist() == list(range(B + 1))
    assert total.tolist() == [c + 1 for c in cached] and pos.tolist() == cached
    want = [(B + i // 3) * P if i % 3 == 0 else i * P + cached[i] for i in range(B)]
    assert slots.tolist() == want
    assert tables[:, 1].tolist() == [B + i // 3 if i % 3 == 0 else -1 for i in range(B)]


def test_page_tables_of_4096_requests_before_any_larger_call():
    """3 * 4 * 4096 bytes of dynamic shared memory are 48 KB, and the kernel's static part comes on top: the first call
    of a process must not rest on a limit that a larger one has raised."""
    code = "import sys; sys.path[:0] = ['', 'tests']; import test_serving_edges_gpu as t; t._decode_tables(4096); print('passed')"
    p = subprocess.run([sys.executable, "-c", code], cwd=ROOT, capture_output=True, text=True, timeout=300)
    assert p.returncode == 0 and "passed" in p.stdout, p.stderr[-2000:]


@pytest.mark.parametrize("B", [4073, 4074, 4096, 4097, 8192, 5000])
def test_page_tables_of_many_requests(B):
    _decode_tables(B)
