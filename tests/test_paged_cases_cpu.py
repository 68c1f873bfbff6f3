"""The measured cases' description of a cache follows the tensors that stand in their state."""
import sys
from pathlib import Path

import pytest

torch = pytest.importorskip("torch")
sys.path.insert(0, str(Path(__file__).resolve().parent.parent / "perf"))


def test_a_caches_description_is_of_the_tensors_that_are_there(monkeypatch):
    import more_operators
    from trs_backend import abi

    monkeypatch.setattr(more_operators, "_backend", lambda: abi)  # no device is asked for

    def tensors():
        return {"pages": [torch.zeros(4, 2, 16, 8) for _ in range(2)], "table": torch.zeros(1, 3, dtype=torch.int32), "lengths": torch.zeros(1, dtype=torch.int32)}

    def described(st):
        c = more_operators._cache(st)
        return (c.k, c.v, c.table, c.lengths, c.table_width, c.type, tuple(c.lk.shape[:4]), tuple(c.lv.stride[:4]))

    def expected(st):
        (k, v), t = st["pages"], st["table"]
        kind = abi.PAGES_BF16 if k.dtype == torch.bfloat16 else abi.PAGES_F32
        return (k.data_ptr(), v.data_ptr(), t.data_ptr(), st["lengths"].data_ptr(), t.shape[1], kind, tuple(k.shape), tuple(v.stride()))

    st = tensors()
    assert described(st) == expected(st) and more_operators._cache(st) is more_operators._cache(st)
    copy = dict(st)
    for key, value in tensors().items():
        copy[key] = value
        assert described(copy) == expected(copy), key
        assert described(st) == expected(st)
    copy["table"] = copy["table"].reshape(3, 1)  # the same memory, read otherwise
    assert described(copy) == expected(copy)
    memory = torch.zeros(4 * 2 * 16 * 8)
    for pool in (memory.view(4, 2, 16, 8), memory.view(4, 2, 8, 16).transpose(2, 3).contiguous(), memory.view(4, 16, 2, 8).transpose(1, 2), memory.view(torch.bfloat16)[:1024].view(4, 2, 16, 8)):
        copy["pages"] = [pool, pool]
        assert described(copy) == expected(copy)
