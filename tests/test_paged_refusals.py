"""What the paged operators refuse, before anything reaches a device."""
from types import SimpleNamespace

import pytest
import torch

from hackthenorth_amd import _lib
from hackthenorth_amd.kernels.paged import (norm_rope_paged, paged_attention,
                                            shared_prefix_attention)

BF16 = torch.bfloat16


def batch(**changes):
    a = dict(q=torch.zeros(3, 4, 128, dtype=BF16), keys=torch.zeros(6, 2, 16, 128, dtype=BF16),
             values=torch.zeros(6, 2, 16, 128, dtype=BF16),
             table=torch.zeros(2, 3, dtype=torch.int32), starts=torch.tensor([0, 1, 3]),
             lengths=torch.tensor([5, 6]))
    a.update(changes)
    return a


def attend(a, **options):
    return paged_attention(a["q"], a["keys"], a["values"], a["table"], a["starts"], a["lengths"],
                           **options)


BAD = [
    (dict(q=torch.zeros(3, 4, 64, dtype=BF16)), "q must be"),
    (dict(q=torch.zeros(3, 4, 128)), "q must be"),
    (dict(q=torch.zeros(3, 128, 4, dtype=BF16).transpose(1, 2)), "q must be"),
    (dict(q=torch.zeros(0, 4, 128, dtype=BF16)), "tokens and heads"),
    (dict(q=torch.zeros(3, 5, 128, dtype=BF16)), "multiple of kv heads"),
    (dict(keys=torch.zeros(6, 2, 24, 128, dtype=BF16), values=torch.zeros(6, 2, 24, 128, dtype=BF16)),
     "power of two"),
    (dict(keys=torch.zeros(6, 2, 8, 128, dtype=BF16), values=torch.zeros(6, 2, 8, 128, dtype=BF16)),
     "power of two"),
    (dict(keys=torch.zeros(6, 2, 2048, 128, dtype=BF16), values=torch.zeros(6, 2, 2048, 128, dtype=BF16)),
     "power of two"),
    (dict(values=torch.zeros(7, 2, 16, 128, dtype=BF16)), "page pools"),
    (dict(values=torch.zeros(6, 2, 16, 128)), "page pools"),
    (dict(keys=torch.zeros(6, 16, 2, 128, dtype=BF16).transpose(1, 2)), "page pools"),
    (dict(table=torch.zeros(2, 3, dtype=torch.int64)), "page_table"),
    (dict(table=torch.zeros(2, 0, dtype=torch.int32)), "page_table"),
    (dict(table=torch.zeros(3, 2, dtype=torch.int32).t()), "page_table"),
    (dict(starts=torch.tensor([0, 3])), "query_starts"),
    (dict(starts=torch.tensor([0, 1, 3], dtype=torch.int32)), "query_starts"),
    (dict(lengths=torch.tensor([5])), "lengths"),
    (dict(lengths=torch.tensor([5.0, 6.0])), "lengths"),
]


@pytest.mark.parametrize("changes,message", BAD)
def test_attention_refuses(changes, message):
    with pytest.raises(ValueError, match=message):
        attend(batch(**changes))
    a = batch(**changes)
    with pytest.raises(ValueError, match=message):
        shared_prefix_attention(a["q"], a["keys"], a["values"], torch.zeros(2, dtype=torch.int32),
                                torch.tensor([4]), a["table"], a["starts"], a["lengths"])


@pytest.mark.parametrize("options,message", [
    (dict(window=-1), "negative"), (dict(window=4, sinks=-2), "negative"), (dict(sinks=3), "window"),
    (dict(out=torch.zeros(3, 4, 128)), "out must"),
    (dict(out=torch.zeros(2, 4, 128, dtype=BF16)), "out must")])
def test_attention_refuses_options(options, message):
    with pytest.raises(ValueError, match=message):
        attend(batch(), **options)


@pytest.mark.parametrize("pages,length", [
    (torch.zeros(2, dtype=torch.int64), torch.tensor([4])), (torch.zeros(0, dtype=torch.int32), torch.tensor([4])),
    (torch.zeros(4, dtype=torch.int32)[::2], torch.tensor([4])),
    (torch.zeros(2, dtype=torch.int32), torch.tensor([4, 5])),
    (torch.zeros(2, dtype=torch.int32), torch.tensor([4], dtype=torch.int32))])
def test_prefix_refuses(pages, length):
    a = batch()
    with pytest.raises(ValueError, match="prefix_"):
        shared_prefix_attention(a["q"], a["keys"], a["values"], pages, length, a["table"], a["starts"],
                                a["lengths"])


def test_cpu_tensors_are_refused():
    a = batch()
    with pytest.raises(ValueError, match="GPU only"):
        attend(a)
    with pytest.raises(ValueError, match="GPU only"):
        append()


def append(**changes):
    norm = SimpleNamespace(weight=torch.ones(128, dtype=BF16), variance_epsilon=1e-6)
    a = batch(q=torch.zeros(3, 4, 128, dtype=BF16), k=torch.zeros(3, 2, 128, dtype=BF16),
              v=torch.zeros(3, 2, 128, dtype=BF16), q_norm=norm, k_norm=norm,
              cos=torch.zeros(9, 128, dtype=BF16), sin=torch.zeros(9, 128, dtype=BF16))
    a.update(changes)
    return norm_rope_paged(a["q"], a["k"], a["v"], a["q_norm"], a["k_norm"], a["cos"], a["sin"],
                           a["keys"], a["values"], a["table"], a["starts"], a["lengths"])


@pytest.mark.parametrize("changes,message", [
    (dict(k=torch.zeros(2, 2, 128, dtype=BF16)), "share"),
    (dict(v=torch.zeros(3, 1, 128, dtype=BF16)), "share"),
    (dict(k=torch.zeros(3, 2, 256, dtype=BF16)[..., :128]), "packed heads"),
    (dict(q=torch.zeros(3, 4, 128)), "q must be"),
    (dict(q_norm=None), "both normalised"),
    (dict(q_norm=SimpleNamespace(weight=torch.ones(64, dtype=BF16), variance_epsilon=0.0)), "gains"),
    (dict(k_norm=SimpleNamespace(weight=torch.ones(128), variance_epsilon=0.0)), "gains"),
    (dict(cos=torch.zeros(9, 64, dtype=BF16), sin=torch.zeros(9, 64, dtype=BF16)), "cos/sin"),
    (dict(cos=torch.zeros(9, 128, dtype=torch.float64), sin=torch.zeros(9, 128, dtype=torch.float64)), "cos/sin"),
    (dict(cos=torch.zeros(9, 128)), "cos/sin"),
    (dict(keys=torch.zeros(6, 3, 16, 128, dtype=BF16), values=torch.zeros(6, 3, 16, 128, dtype=BF16)),
     "page pools"),
    (dict(table=torch.zeros(2, 3)), "page_table")])
def test_append_refuses(changes, message):
    with pytest.raises(ValueError, match=message):
        append(**changes)


def test_library_checks_before_any_launch():
    lib, p = _lib.load(), 4096

    def paged(**c):
        a = dict(q=p, q_st=512, q_sh=128, page=16, table_pages=3, window=0, sinks=0, out=p, o_st=512,
                 batch=2, tokens=3, heads=4, kv=2, scratch=p, size=1 << 30)
        a.update(c)
        return lib.htn_paged_attention(a["q"], a["q_st"], a["q_sh"], p, p, 6, a["page"], p, 3, a["table_pages"],
                                       p, p, a["window"], a["sinks"], a["out"], a["o_st"], 128, a["batch"],
                                       a["tokens"], a["heads"], a["kv"], a["scratch"], a["size"], None)
    assert paged(q=None) == _lib.HTN_EINVAL and paged(scratch=None) == _lib.HTN_EINVAL
    assert paged(page=20) == _lib.HTN_EINVAL and paged(heads=5) == _lib.HTN_EINVAL
    assert paged(window=-1) == _lib.HTN_EINVAL and paged(sinks=-1) == _lib.HTN_EINVAL
    assert paged(size=1 << 10) == _lib.HTN_EINVAL and paged(batch=0) == _lib.HTN_EINVAL
    assert paged(q=p + 2) == _lib.HTN_EUNSUPPORTED and paged(q_st=516) == _lib.HTN_EUNSUPPORTED
    assert paged(o_st=514) == _lib.HTN_EUNSUPPORTED and paged(out=p + 4) == _lib.HTN_EUNSUPPORTED
    assert paged(table_pages=1 << 26) == _lib.HTN_EUNSUPPORTED
    assert paged(tokens=1 << 31) == _lib.HTN_EUNSUPPORTED
    assert lib.htn_paged_attention_scratch_bytes(3, 2, 4, 2, 0) > 0
    assert lib.htn_paged_attention_scratch_bytes(3, 2, 5, 2, 0) == 0
