"""What sample_token refuses, before anything reaches a device."""
import pytest
import torch

from hackthenorth_amd import _lib
from hackthenorth_amd.kernels.sample import sample_token

LOGITS, U = torch.zeros(3, 10), torch.zeros(3)


@pytest.mark.parametrize("logits,uniform,settings,message", [
    (LOGITS.half(), U, {}, "bf16 or fp32"), (torch.zeros(()), U[:1], {}, "bf16 or fp32"),
    (torch.zeros(0, 10), U[:0], {}, "bf16 or fp32"), (torch.zeros(3, 0), U, {}, "bf16 or fp32"),
    (LOGITS, U[:2], {}, "uniform"), (LOGITS, U.double(), {}, "uniform"),
    (LOGITS, torch.zeros(6)[::2], {}, "uniform"),
    (LOGITS, U, dict(temperature=-0.1), "temperature"), (LOGITS, U, dict(temperature=float("nan")), "temperature"),
    (LOGITS, U, dict(temperature=torch.ones(2)), "temperature"),
    (LOGITS, U, dict(temperature=torch.ones(3, dtype=torch.float64)), "temperature"),
    (LOGITS, U, dict(top_k=-1), "top_k"), (LOGITS, U, dict(top_k=torch.ones(3)), "top_k"),
    (LOGITS, U, dict(top_p=-0.5), "top_p"), (LOGITS, U, dict(min_p=float("nan")), "min_p"),
    (LOGITS, U, dict(out=torch.zeros(3)), "out"), (LOGITS, U, dict(out=torch.zeros(2, dtype=torch.int64)), "out"),
    (LOGITS, U, {}, "GPU only")])
def test_refuses(logits, uniform, settings, message):
    with pytest.raises(ValueError, match=message):
        sample_token(logits, uniform, **settings)


def test_library_checks_before_any_launch():
    lib, p = _lib.load(), 4096

    def sample(**c):
        a = dict(logits=p, st=10, fp32=1, rows=3, vocab=10, uniform=p, out=p, scratch=p, size=1 << 20)
        a.update(c)
        return lib.htn_sample(a["logits"], a["st"], a["fp32"], a["rows"], a["vocab"], a["uniform"], None, 1.0,
                              None, 0, None, 1.0, None, 0.0, a["out"], a["scratch"], a["size"], None)
    for bad in (dict(logits=None), dict(uniform=None), dict(out=None), dict(scratch=None), dict(rows=0),
                dict(vocab=0), dict(st=9), dict(size=100)):
        assert sample(**bad) == _lib.HTN_EINVAL
    for bad in (dict(rows=65536), dict(vocab=(1 << 19) + 1, st=1 << 20), dict(logits=p + 2), dict(scratch=p + 8)):
        assert sample(**bad) == _lib.HTN_EUNSUPPORTED
    assert lib.htn_sample_scratch_bytes(3, 10) > 0 and lib.htn_sample_scratch_bytes(0, 10) == 0
