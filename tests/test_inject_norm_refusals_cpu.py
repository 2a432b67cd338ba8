"""What ``inject_norm`` and its gradients answer on the host, before any launch."""
import pytest
import torch


def lib():
    import build as fnx_build
    fnx_build.build()
    from fnx import _lib
    return _lib.lib()


@pytest.mark.parametrize("H,HC", [(512, 1), (4096, 1), (4104, 1), (1864, 2), (2048, 2), (2560, 2), (1536, 3), (2048, 3),
                                  (1288, 4), (2048, 4), (4104, 4)])
def test_the_backward_launches_no_more_blocks_than_fit(H, HC):
    """Its blocks are persistent: one that does not fit waits for another to end and then starts its copies
    anew, and each writes its own partial sums.  The kernels' launch bounds (512 threads, one block an SM;
    two for one branch of H <= 4096) let the compiler take 65536 / 512 = 128 registers a thread, or 64."""
    sms = torch.cuda.get_device_properties(0).multi_processor_count if torch.cuda.is_available() else 148
    blocks, rest = divmod(lib().fnx_inject_norm_backward_workspace(1 << 20, H, HC), (HC + 1) * H * 4)
    threads = (H // 8 + 31) // 32 * 32 if H <= 4096 else 512
    registers = 64 if HC == 1 and H <= 4096 else 128
    assert rest == 0 and blocks % sms == 0
    assert 1 <= blocks // sms <= max(1, 65536 // (registers * threads))
