"""What the operators for drafted tokens refuse before they look for a GPU: no tensors, tensors on the CPU, no cache."""
import pytest
import torch

from vdcores_b200 import ops


@pytest.mark.parametrize("logits", [None, [1.0, 2.0], "logits", torch.zeros(2, 8), torch.zeros(8), torch.zeros(2, 8, dtype=torch.int32)])
def test_logits_that_are_none(logits):
    for _ in range(2):
        with pytest.raises(ValueError):
            ops.adjust_logits(logits)


def test_tables_that_are_none():
    with pytest.raises(ValueError):
        ops.adjust_logits(torch.zeros(1, 8), history=[[1, 2]], repetition=[1.0])


def test_no_cache():
    x, i = torch.zeros(1, 1, 4, 128, dtype=torch.bfloat16), torch.zeros(1, dtype=torch.int32)
    for call in (lambda: ops.rope_append(x, x, x, None, i[None], i), lambda: ops.tree_attention(x, (x, x), i[None], i),
                 lambda: ops.read_cache(None, i[None], i, 4)):
        with pytest.raises(ValueError, match="KVCache"):
            call()
    with pytest.raises(ValueError):
        ops.KVCache(torch.zeros(2, 1, 64, 128, dtype=torch.bfloat16), torch.zeros(2, 1, 64, 128, dtype=torch.bfloat16))


def test_a_site_takes_its_number_of_arguments():
    with pytest.raises(TypeError):
        ops._adjust(b"", ())
    with pytest.raises(TypeError):
        ops._adjust("", (), *[None] * 13)
