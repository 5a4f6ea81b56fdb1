"""Calls of the distillation operator by several host threads at once."""
import ctypes
import threading

import pytest
import torch

pytestmark = pytest.mark.gpu


def test_distill_calls_of_different_sizes_by_threads():
    """Launches that need different amounts of dynamic shared memory (41, 47 and 52 KB), each thread on a stream of its own: no
    call may fail for what another one asks for."""
    from xlstm_b200 import _lib
    l = _lib.lib()
    K, errors, keep, args = 1024, [], [], []
    for V in (165000, 210000, 2 ** 18):
        x = torch.zeros(1, V, dtype=torch.bfloat16, device="cuda")
        values, ids = torch.zeros(1, K, device="cuda"), torch.arange(K, dtype=torch.int32, device="cuda")[None]
        loss, dx, stream = torch.zeros(1, device="cuda"), torch.empty(300, V, dtype=torch.bfloat16, device="cuda"), torch.cuda.Stream()
        p = _lib.DistillParams()
        x = x.expand(300, V).contiguous()   # (more rows than are cut over blocks)
        values, ids, loss = values.expand(300, K).contiguous(), ids.expand(300, K).contiguous(), loss.expand(300).contiguous()
        p.logits, p.values, p.ids, p.loss, p.dlogits = (t.data_ptr() for t in (x, values, ids, loss, dx))
        p.rows, p.V, p.K, p.row_stride, p.dlogits_stride, p.cap, p.temperature, p.dtype = 300, V, K, V, V, 30.0, 1.0, 1
        keep.append((x, values, ids, loss, dx, stream))
        args.append((p, stream.cuda_stream))
    torch.cuda.synchronize()

    def work(p, stream):
        device = torch.cuda.current_device()
        torch.cuda.set_device(device)
        for _ in range(300):
            rc = l.xl_distill_topk(ctypes.byref(p), stream)
            if rc:
                errors.append(rc)
    threads = [threading.Thread(target=work, args=a) for a in args]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    torch.cuda.synchronize()
    assert not errors
    for x, values, ids, loss, dx, stream in keep:
        want = torch.tensor(x.shape[1] / K).log()          # all logits equal, the teacher flat over K tokens
        assert (loss.cpu() - want).abs().max() < 1e-5
