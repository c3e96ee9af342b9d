"""The gated residual and adaptive RMS norm (bf16) with the new residual written over the old one, which the C entry allows."""
import ctypes

import pytest
import torch

from krea2_svdquant_amd.kernels.hip import lib, ops


@pytest.mark.skipif(not lib.LIB_PATH.exists(), reason="library not built")
def test_another_stride_in_place_is_refused():
    p, q = ctypes.c_void_p(0x1000), ctypes.c_void_p(0x2000)   # never read: the call fails on the host
    with pytest.raises(lib.SVDQError, match="ldxo") as e:
        lib.call("svdq_residual_rms_norm_modulate", p, 64, q, 64, q, q, q, 2, 64, ctypes.c_float(0), p, 72, q, 64, None)
    assert e.value.status == -2


@pytest.mark.gpu
@pytest.mark.parametrize("m,h,ld", [(1, 8, 8), (70, 512, 520), (300, 6144, 6144), (9, 20000, 20008)])
def test_in_place(dev, m, h, ld):
    gen = torch.Generator(device=dev).manual_seed(m)
    buf, v, gate, w, shift = (torch.randn(s, device=dev, generator=gen).to(torch.bfloat16)
                              for s in ((m, ld), (m, h), (h,), (h,), (h,)))
    want, want_y = ops.residual_rms_norm_modulate(buf[:, :h], v, gate, w, shift, 1e-6)
    behind, y = buf[:, h:].clone(), torch.empty(m, h, device=dev, dtype=torch.bfloat16)
    lib.call("svdq_residual_rms_norm_modulate", buf.data_ptr(), ld, v.data_ptr(), h, gate.data_ptr(), w.data_ptr(),
             shift.data_ptr(), m, h, 1e-6, buf.data_ptr(), ld, y.data_ptr(), h, torch.cuda.current_stream().cuda_stream)
    assert torch.equal(buf[:, :h], want) and torch.equal(y, want_y) and torch.equal(buf[:, h:], behind)
