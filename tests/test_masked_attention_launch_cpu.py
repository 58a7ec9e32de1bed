"""Host side of the masked attention launchers against the fake CUDA runtime, and of their workspaces, on the CPU."""
import ctypes

import pytest
from test_launchers_cpu import BUF, fake  # noqa: F401

from gpt_from_scratch_b200.ops import _lib
from gpt_from_scratch_b200.ops.masked_attention import _scratch


def backward(lib, partial, floats, S=300, B=1, nh=8, nkv=1, D=64):
    strides = (ctypes.c_longlong * 24)(*[D, D * S * nh, D * S] * 8)
    return lib.gfs_masked_attention_bwd(*[BUF] * 7, partial, floats, *[BUF] * 4, S, B, nh, nkv, D, strides, 0.1, 0.0, 0, 0)


def test_the_backward_refuses_too_little_scratch(fake):  # noqa: F811
    """The number of parts follows from the device's SMs, so a size that another device gave may be too small."""
    need = fake.gfs_masked_attention_scratch(300, 1, 8, 1, 64)
    assert need == 2 * 4 * 3 * 128 * 64
    for partial, floats in ((BUF, need - 1), (BUF, 0), (0, 0), (0, need), (BUF + 4, need)):
        before = fake.fake_launches()
        assert backward(fake, partial, floats) != 0 and fake.fake_launches() == before
    assert backward(fake, BUF, need) == 0 and backward(fake, BUF, need + 1) == 0
    assert fake.gfs_masked_attention_scratch(300, 64, 8, 8, 64) == 0 and backward(fake, 0, 0, B=64, nkv=8) == 0


def test_scratch_sizes_belong_to_a_device(monkeypatch):
    class Library:
        sms = 0

        def gfs_masked_attention_scratch(self, *sizes):
            return self.sms
    lib = Library()
    monkeypatch.setattr(_lib, "lib", lambda: lib)
    sizes = (301, 7, 8, 1, 64)
    for device, sms in ((0, 148), (1, 64)):
        lib.sms = sms
        assert _scratch(*sizes, device) == sms
    _scratch.cache_clear()


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("cap,slopes", [(0.0, 0), (30.0, 0), (900.0, 0), (30.0, BUF), (0.0, BUF)])
def test_every_device_of_a_process_is_served(fake, D, cap, slopes):  # noqa: F811
    """As for the other kernels: the limit on dynamic shared memory is raised on each device."""
    strides = (ctypes.c_longlong * 24)(*[D, D * 300 * 8, D * 300] * 8)
    for dev in (0, 1, 0, 2):
        fake.fake_set_device(dev)
        assert fake.gfs_masked_attention_fwd(*[BUF] * 6, 300, 1, 8, 8, D, strides, 0.1, cap, slopes, 0) == 0
        assert fake.gfs_masked_attention_bwd(*[BUF] * 8, 1 << 30, *[BUF] * 4, 300, 1, 8, 8, D, strides, 0.1, cap, slopes, 0) == 0
    fake.fake_set_device(0)


def test_entries_refuse_what_would_end_the_process(fake):  # noqa: F811
    """No key heads (a division), no place for what a kernel writes."""
    for sizes in ((300, 1, 8, 0, 64), (300, 1, 0, 0, 64), (0, 1, 8, 1, 64), (-5, 1, 8, 1, 64)):
        assert fake.gfs_masked_attention_scratch(*sizes) == 0
    before = fake.fake_launches()
    strides = (ctypes.c_longlong * 24)(*[64, 64 * 300 * 8, 64 * 300] * 8)
    for hole in (5, 6, 11):             # saved, dvec, mask
        at = [0 if i == hole else BUF for i in range(12)]
        assert fake.gfs_masked_attention_bwd(*at[:8], 1 << 30, *at[8:], 300, 1, 8, 8, 64, strides, 0.1, 0.0, 0, 0) != 0
    assert fake.gfs_masked_attention_fwd(*[BUF] * 5, 0, 300, 1, 8, 8, 64, strides, 0.1, 0.0, 0, 0) != 0
    assert fake.gfs_attention_mask(0, 0, 0, 1, 300, 1, 0, 0, 0) != 0
    for hole in range(3):               # the weights' gradients and their scratch
        dw = [0 if i == hole else BUF for i in range(3)]
        assert fake.gfs_qk_norm_rope_bwd(*[BUF] * 5, strides, BUF, BUF, *dw, BUF, BUF, 0, 0, 300, 300, 1, 4, 2, 64, 64, 0, 1e-5, 0, 0) != 0
    assert fake.fake_launches() == before
