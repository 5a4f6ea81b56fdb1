"""Host side of the vocabulary operators: parameter blocks, checks in front of every launch, refusals (no GPU)."""
import ctypes
import os
import re

import pytest
import torch

from conftest import ROOT


def test_parameter_blocks_match_the_header():
    from xlstm_b200 import _lib
    header = open(os.path.join(ROOT, "include", "xlstm_b200.h")).read()
    for cname, struct in (("xl_sample_params", _lib.SampleParams), ("xl_topk_params", _lib.TopkParams), ("xl_distill_params", _lib.DistillParams)):
        body = re.search(r"typedef struct %s \{(.*?)\} %s;" % (cname, cname), header, re.S).group(1)
        body = re.sub(r"/\*.*?\*/", "", body, flags=re.S)
        names = []
        for decl in filter(None, (d.strip() for d in body.split(";"))):
            first, *rest = decl.split(",")
            names += [re.findall(r"[A-Za-z_0-9]+", d)[-1] for d in (first, *rest)]
        assert names == [f[0] for f in struct._fields_], cname


def test_entries_check_before_they_launch():
    from xlstm_b200 import _lib
    l = _lib.lib()
    ref = ctypes.byref
    s = _lib.SampleParams()
    assert l.xl_softcap_sample(ref(s), None) == -1
    s.logits = s.tokens = s.u = 0x1000
    s.rows, s.V, s.row_stride, s.dtype = 2, 8, 8, 2
    assert l.xl_softcap_sample(ref(s), None) == -5      # no such type
    s.dtype, s.V = 1, 0
    assert l.xl_softcap_sample(ref(s), None) == -2
    s.V, s.cap = 8, -1.0
    assert l.xl_softcap_sample(ref(s), None) == -2      # negative cap
    s.cap, s.row_stride = 0.0, 7
    assert l.xl_softcap_sample(ref(s), None) == -3      # rows overlap
    s.V = s.row_stride = 2 ** 18 + 1
    assert l.xl_softcap_sample(ref(s), None) == -8
    t = _lib.TopkParams()
    assert l.xl_softcap_topk(ref(t), None) == -1
    t.logits = t.values = t.ids = 0x1000
    t.rows, t.V, t.row_stride, t.dtype, t.k = 2, 8, 8, 1, 9
    assert l.xl_softcap_topk(ref(t), None) == -2        # k above V
    t.k = 8
    assert l.xl_softcap_topk(ref(t), None) == -2        # no temperature
    t.temperature, t.V, t.row_stride, t.k = 1.0, 2048, 2048, 1025
    assert l.xl_softcap_topk(ref(t), None) == -8
    d = _lib.DistillParams()
    for entry in (l.xl_distill_topk, l.xl_distill_topk_backward):
        assert entry(ref(d), None) == -1
    d.logits, d.values, d.ids, d.loss = 0x1000, 0x2000, 0x3000, 0x4000
    d.rows, d.V, d.row_stride, d.dtype, d.K, d.temperature = 2, 8, 8, 1, 0, 1.0
    assert l.xl_distill_topk(ref(d), None) == -2        # no entries
    d.K = 1025
    assert l.xl_distill_topk(ref(d), None) == -8
    d.K = 2
    assert l.xl_distill_topk_backward(ref(d), None) == -1   # neither stats nor dlogits
    d.dlogits, d.dlogits_stride = 0x1010, 8
    assert l.xl_distill_topk(ref(d), None) == -9        # the gradient over the logits of the second row
    d.dlogits, d.dlogits_stride = 0x8000, 4
    assert l.xl_distill_topk(ref(d), None) == -3
    d.dlogits_stride, d.loss = 8, None
    assert l.xl_distill_topk(ref(d), None) == -1


def test_operators_refuse_host_tensors():
    import xlstm_b200
    x, u = torch.zeros(2, 8), torch.zeros(2)
    ids = torch.zeros(2, 3, dtype=torch.int32)
    for call in (lambda: xlstm_b200.softcap_sample(x, 30.0, u), lambda: xlstm_b200.softcap_topk(x, 30.0, 2),
                 lambda: xlstm_b200.distill_topk(x, u, ids), lambda: xlstm_b200.distill_topk_grad(x, u, ids),
                 lambda: xlstm_b200.distill_topk(x.requires_grad_(), u, ids)):
        with pytest.raises(ValueError, match="no CPU path"):
            call()
    with pytest.raises(ValueError, match="temperature"):
        xlstm_b200.softcap_sample(x, 30.0, u, temperature=-1.0)
    with pytest.raises(ValueError, match="cap"):
        xlstm_b200.softcap_topk(x, 0.0, 2)


def test_entries_refuse_addresses_inside_an_element():
    from xlstm_b200 import _lib
    l = _lib.lib()
    for dtype, off in ((0, 1), (0, 2), (1, 1)):
        s, t, d = _lib.SampleParams(), _lib.TopkParams(), _lib.DistillParams()
        for p in (s, t, d):
            p.logits, p.rows, p.V, p.row_stride, p.dtype, p.temperature = 0x1000 + off, 2, 8, 8, dtype, 1.0
        s.tokens = s.u = 0x2000
        t.values = t.ids = d.values = d.ids = d.loss = 0x2000
        t.k = d.K = 2
        assert l.xl_softcap_sample(ctypes.byref(s), None) == -4
        assert l.xl_softcap_topk(ctypes.byref(t), None) == -4
        assert l.xl_distill_topk(ctypes.byref(d), None) == -4
        d.logits, d.dlogits, d.dlogits_stride, d.stats = 0x1000, 0x8000 + off, 8, 0x9000
        for entry in (l.xl_distill_topk, l.xl_distill_topk_backward):
            assert entry(ctypes.byref(d), None) == -4
