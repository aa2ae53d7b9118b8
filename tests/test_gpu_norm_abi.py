"""Residual norm through the C ABI: what it is asked for that does not depend on what it is given."""
import ctypes

import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("bs_last", [0, 1])
@pytest.mark.parametrize("features,batch", [(40, 30), (1300, 30)])
def test_parameters_of_an_output_without_gradient(features, batch, bs_last, lib):
    """dn_out NULL is a gradient of zeros: so are those of the last norm's weight and bias, through the C ABI too."""
    from ksmm_amd._lib import KsmmNormDesc

    for dt in (torch.float32, torch.float16):
        shape = (features, batch) if bs_last else (batch, features)
        x, r, dr = (torch.randn(shape, device="cuda").to(dt) for _ in range(3))
        w, b = torch.ones(features, device="cuda").to(dt), torch.ones(features, device="cuda").to(dt)
        code = 0 if dt == torch.float32 else 1
        desc = KsmmNormDesc(x.data_ptr(), r.data_ptr(), None, None, w.data_ptr(), b.data_ptr(), 1, 0.5, 1e-6, 0)
        out, n, stats = torch.empty_like(r), torch.empty_like(r), torch.empty(4, batch, device="cuda")
        ws = torch.empty(max(16, lib.ksmm_residual_norm_forward_workspace(batch, features, code, bs_last)), dtype=torch.uint8, device="cuda")
        stream = ctypes.c_void_p(torch.cuda.current_stream().cuda_stream)
        assert lib.ksmm_residual_norm_forward(ctypes.byref(desc), out.data_ptr(), n.data_ptr(), stats.data_ptr(), ws.data_ptr(), ws.numel(), batch,
                                              features, code, bs_last, stream) == 0
        need = lib.ksmm_residual_norm_backward_workspace(batch, features, 1, code, bs_last)
        ws = torch.empty(need, dtype=torch.uint8, device="cuda")
        for which in ((1, 1), (1, 0), (0, 1)):
            dx, dw, db = torch.empty_like(x), torch.full_like(w, 7.0), torch.full_like(b, 7.0)
            assert lib.ksmm_residual_norm_backward(ctypes.byref(desc), stats.data_ptr(), dr.data_ptr(), None, dx.data_ptr(), None, None, None,
                                                   dw.data_ptr() if which[0] else None, db.data_ptr() if which[1] else None, ws.data_ptr(), need, batch,
                                                   features, code, bs_last, stream) == 0
            torch.cuda.synchronize()
            assert torch.equal(dx, (dr.float() * 0.5).to(dt))
            assert bool(dw.any()) == (not which[0]) and bool(db.any()) == (not which[1])
