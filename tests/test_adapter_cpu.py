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


def test_products_that_may_overlap_share_no_scratch(monkeypatch):
    """A generation-step product keeps arrival counters and partial sums in its scratch: calls on two streams, and captured calls, have their own."""
    from energonai_b200 import adapter, gemm
    L = _lib.lib()
    # few rows of a large weight count, the step form of a small one and tiles of 128 rows do not
    assert L.eb_gemm_counter_bytes(16, 5120, 5120, 5120) == 40 * 16 and L.eb_gemm_counter_bytes(40, 520, 512, 516) == 5 * 16
    assert L.eb_gemm_counter_bytes(16, 1024, 1024, 1024) == 0 and L.eb_gemm_counter_bytes(48, 5120, 5120, 5120) == 0 and L.eb_gemm_counter_bytes(200, 5120, 5120, 5120) == 0
    stream, capturing = [7], [False]
    monkeypatch.setattr(gemm, "stream_ptr", lambda: stream[0])
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: capturing[0])
    monkeypatch.setattr(gemm, "_stream_workspaces", {})
    large = lambda: gemm.stream_workspace("cpu", 16, 5120, 5120, 5120)
    first, again = large(), large()
    assert first is again and first.numel() >= L.eb_gemm_workspace_bytes(16, 5120, 5120) and not first.any()
    assert gemm.stream_workspace("cpu", 32, 5120, 5120, 5120).numel() > first.numel()
    stream[0] = 9
    other = large()
    assert other.data_ptr() != first.data_ptr()
    capturing[0] = True
    captured = [large() for _ in range(2)]
    assert len({t.data_ptr() for t in (first, other, *captured)}) == 4 and all(not t[:640].any() for t in captured)
    assert gemm.stream_workspace("cpu", 200, 5120, 5120, 5120) is None

    # ... and adapter_product asks for it
    asked = []
    monkeypatch.setattr(adapter, "_one_device", lambda *a: 0)
    monkeypatch.setattr(adapter, "adapter_delta", lambda *a: None)
    monkeypatch.setattr(adapter, "gemm", lambda *a, **kw: asked.append(kw))
    adapter.adapter_product(torch.zeros(2, 64), torch.zeros(16, 64), torch.zeros(1, 8, 64), torch.zeros(1, 16, 8), None, None, None, 2)
    assert asked[0]["overlap"] is True


def test_the_two_launches_refuse():
    of = dict(x=FAKE, ldx=64, a=FAKE)
    sequences = dict(index=FAKE, starts=FAKE)
    sizes = dict(rank=16, adapters=3, batch=2, most_new=4, dtype=_lib.F16, scratch=FAKE, scratch_bytes=1 << 20, stream=None)
    low = {**of, **sequences, "rows": 4, "width": 64, **sizes}
    add = {"b": FAKE, "scales": FAKE, **sequences, "base": FAKE, "ldbase": 128, "out": FAKE, "ldo": 128, "rows": 4, "width": 64, "columns": 128, **sizes}
    L = _lib.lib()
    both = [(dict(index=None), "null"), (dict(dtype=_lib.BF16), "fp16 only"), (dict(dtype=_lib.F32), "fp16 or bf16"), (dict(rank=12), "rank 12"), (dict(scratch_bytes=8), "scratch"),
            (dict(most_new=0), "bad sizes"), (dict(batch=0), "bad sizes")]
    for change, words in both + [(dict(x=None), "null"), (dict(a=FAKE + 8), "16-byte"), (dict(ldx=56), "hold a row"), (dict(width=60), "multiples of 8")]:
        assert L.eb_adapter_low(*{**low, **change}.values()) == -1 and words in _lib.last_error(), change
    for change, words in both + [(dict(base=None), "null"), (dict(out=None), "null"), (dict(ldbase=124), "hold a row"), (dict(ldbase=120), "hold a row"), (dict(ldo=132), "hold a row"),
                                 (dict(base=FAKE + 4), "16-byte"), (dict(columns=124), "multiples of 8")]:
        assert L.eb_adapter_add(*{**add, **change}.values()) == -1 and words in _lib.last_error(), change
    assert L.eb_adapter_low(*{**low, "rows": 0}.values()) == 0 and L.eb_adapter_add(*{**add, "rows": 0}.values()) == 0
