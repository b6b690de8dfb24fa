"""What packing a 4-bit weight reports, and to whom."""
import threading

import pytest

from test_q4_gpu import check, product, weights

pytestmark = pytest.mark.gpu


def test_reports_of_other_calls_stay_theirs(cuda):
    """A dispatch's bad expert id is neither the weight's nor lost to it; a weight's
    bad value is raised by its own call and left nowhere else."""
    import torch
    from aethermoe_b200 import _lib, q4
    from aethermoe_b200 import dispatch as D
    q, s = weights(cuda, 1, 200, 40, 64, torch.float32)
    bad = q.clone()
    bad[0, 199, 39] = 8
    assert _lib.lib().aem_device_status(None) == _lib.AEM_OK
    ids = torch.full((4, 1), 9, dtype=torch.int32, device=cuda)
    D.sort_tokens(ids, 4)
    w = q4.Q4Weight(q, s, 64)
    with pytest.raises(ValueError, match="-7, 7"):
        q4.Q4Weight(bad, s, 64)
    x = torch.randn(3, 200, device=cuda)
    ref, A = product(x, q[0], s[0], 64)
    check(q4.q4_matmul(x, w), ref, A, 4)
    assert _lib.lib().aem_device_status(None) == _lib.AEM_EDEVICE
    assert "expert id" in _lib.last_error() and "4-bit" not in _lib.last_error()
    assert _lib.lib().aem_device_status(None) == _lib.AEM_OK


def test_bad_values_beside_another_threads_status_calls(cuda):
    """Threads that pack good and bad weights while others read and clear the shared
    word: every bad weight raises and no good one does."""
    import torch
    from aethermoe_b200 import _lib, q4
    q, s = weights(cuda, 2, 512, 256, 128, torch.bfloat16)
    bad = q.clone()
    bad[1, 300, 200] = -8
    said = [[], []]

    def pack(i):
        with torch.cuda.stream(torch.cuda.Stream()):
            for _ in range(40):
                try:
                    q4.Q4Weight(bad if i else q, s, 128).close()
                    said[i].append("packed")
                except ValueError as e:
                    said[i].append("refused" if "-7, 7" in str(e) else str(e))

    over = threading.Event()
    states = set()

    def status():
        side = torch.cuda.Stream()
        with torch.cuda.device(cuda):
            while not over.is_set():
                states.add(_lib.lib().aem_device_status(side.cuda_stream))
    threads = [threading.Thread(target=pack, args=(i,)) for i in range(2)]
    reader = threading.Thread(target=status)
    torch.cuda.synchronize()
    reader.start()
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    over.set()
    reader.join()
    assert said == [["packed"] * 40, ["refused"] * 40] and states == {_lib.AEM_OK}


def test_stream_ordered_pack_reports_in_the_shared_word(cuda):
    """The C form that does not wait clamps and leaves its report to the device's status."""
    import ctypes
    import torch
    from aethermoe_b200 import _lib
    q, s = weights(cuda, 1, 128, 64, 64, torch.float32)
    h = ctypes.c_void_p()
    st = torch.cuda.current_stream().cuda_stream
    for value, want in ((7, _lib.AEM_OK), (12, _lib.AEM_EDEVICE)):
        q[0, 5, 6] = value
        assert _lib.lib().aem_q4weight_pack_device(q.data_ptr(), s.data_ptr(), _lib.F32, 1, 128, 64, 64, st,
                                                   ctypes.byref(h)) == _lib.AEM_OK
        assert _lib.lib().aem_device_status(st) == want
        _lib.lib().aem_q4weight_free(h)
    assert _lib.lib().aem_q4weight_pack_checked(q.data_ptr(), s.data_ptr(), _lib.F32, 1, 128, 64, 64, st,
                                                ctypes.byref(h)) == _lib.AEM_EINVAL and not h.value
    assert _lib.lib().aem_device_status(st) == _lib.AEM_OK


def test_packing_refuses_tensors_of_two_devices(cuda):
    import torch
    from aethermoe_b200 import q4
    q, s = weights(cuda, 1, 64, 32, 32, torch.float32)
    for a, b in ((q.cpu(), s), (q, s.cpu())):
        with pytest.raises(ValueError, match="one CUDA device or the CPU"):
            q4.Q4Weight(a, b, 32)


def test_host_pack_keeps_the_current_device(cuda):
    import torch
    from aethermoe_b200 import q4
    if torch.cuda.device_count() < 2:
        pytest.skip("needs two devices")
    q, s = weights(cuda, 1, 64, 32, 32, torch.float32)
    w = q4.Q4Weight(q[0].cpu(), s[0].cpu(), 32, device=1)
    assert torch.cuda.current_device() == 0 and w.device == 1
    x = torch.randn(2, 64, device="cuda:1")
    assert torch.equal(q4.q4_matmul(x, w).cpu(), q4.q4_matmul(x.to(cuda), q4.Q4Weight(q[0], s[0], 32)).cpu())
    assert torch.cuda.current_device() == 0
