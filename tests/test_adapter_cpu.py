"""Low-rank adapters: what is refused before anything runs."""
import pytest
import torch

from energonai_b200 import _lib

FAKE = 1 << 20                 # an aligned address that nothing is read from: every call below is refused before a launch


def call(**change):
    a = dict(x=FAKE, ldx=64, a=FAKE, b=FAKE, scales=FAKE, index=FAKE, starts=FAKE, delta=FAKE, ldd=128, rows=4, width=64, columns=128, rank=16, adapters=3, batch=2,
             most_new=4, dtype=_lib.BF16, scratch=FAKE, scratch_bytes=1 << 20, stream=None)
    a.update(change)
    return _lib.lib().eb_adapter_delta(*a.values())


@pytest.mark.parametrize("change,words", [(dict(x=None), "null"), (dict(starts=None), "null"), (dict(dtype=_lib.F32), "fp16 or bf16"), (dict(rank=12), "rank 12"), (dict(rank=0), "rank 0"),
                                          (dict(rank=136), "rank 136"), (dict(width=60), "multiples of 8"), (dict(ldx=56), "hold a row"), (dict(ldd=120), "hold a row"),
                                          (dict(columns=124), "multiples of 8"), (dict(a=FAKE + 8), "16-byte"), (dict(scratch=None), "scratch"), (dict(scratch_bytes=8), "scratch"),
                                          (dict(batch=0), "bad sizes"), (dict(most_new=0), "bad sizes"), (dict(adapters=0), "bad sizes")])
def test_delta_refuses(change, words):
    assert call(**change) == -1 and words in _lib.last_error()


def test_nothing_to_do():
    assert call(rows=0) == 0 and call(columns=0) == 0
    assert _lib.lib().eb_adapter_scratch_bytes(0, 64, 16, 2, 4) == 0


def test_cpu_tensors_are_rejected():
    from energonai_b200.adapter import adapter_delta, adapter_product
    x, a, b = torch.zeros(2, 64), torch.zeros(1, 8, 64), torch.zeros(1, 16, 8)
    i32 = lambda v: torch.tensor(v, dtype=torch.int32)
    with pytest.raises(RuntimeError, match="CUDA"):
        adapter_delta(x, a, b, torch.ones(1), i32([0]), i32([0, 2]), 2)
    with pytest.raises(RuntimeError, match="CUDA"):
        adapter_product(x, torch.zeros(16, 64), a, b, torch.ones(1), i32([0]), i32([0, 2]), 2)
