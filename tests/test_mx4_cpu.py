"""Microscaled 4-bit row products on the host: the format's plain statement, argument checks of the C entries and of the
Python functions (nothing here launches a kernel)."""
import ctypes as C

import numpy as np
import pytest
import torch

from tests import _mx4_ref as ref


def test_plain_statement_of_the_format():
    x = np.zeros((1, 32))
    x[0, :12] = [4.0, 0.25, 0.26, 0.75, 1.25, 1.75, 2.5, 3.5, -5.0, 5.01, 7.9, -0.1]       # top in [4, 8): scale 1
    codes, scales = ref.round_codes(x)
    assert scales[0, 0] == 127 and scales[0, 1:].tolist() == [0] * 7
    assert codes[0, :12].tolist() == [6, 0, 1, 2, 2, 4, 4, 6, 8 + 6, 7, 7, 8]
    assert ref.code_values(codes, scales, 12).tolist() == [[4, 0, .5, 1, 1, 2, 2, 4, -4, 6, 6, 0]]
    for bad in (np.inf, -np.inf, np.nan):
        y = np.ones((1, 40))
        y[0, 3] = bad
        v = ref.code_values(*ref.round_codes(y), 40)
        assert np.isnan(v[0, :32]).all() and (v[0, 32:] == 1).all()
    tiny = np.full((1, 3), 2.0 ** -140)
    assert ref.round_codes(tiny)[1][0, 0] == 0


def test_entries_check_their_arguments():
    from sln_amodal_amd import _lib
    L = _lib.lib()
    buf = (C.c_char * 4096)()
    p = C.c_void_p((C.addressof(buf) + 255) // 256 * 256)
    odd = C.c_void_p(p.value + 1)
    INVALID, WORKSPACE, UNSUPPORTED = 1, 2, 4
    assert [L.sln_mx4_row_values(k) for k in (0, 1, 256, 257, 12544)] == [0, 256, 256, 512, 12544]
    assert L.sln_mx4_round(p, 3, 1, 1, 1, p, p, None) == INVALID
    assert L.sln_mx4_round(p, 0, 1, 0, 1, p, p, None) == INVALID
    assert L.sln_mx4_round(p, 0, -1, 4, 4, p, p, None) == INVALID
    assert L.sln_mx4_round(p, 0, 2, 4, 3, p, p, None) == INVALID
    assert L.sln_mx4_round(p, 0, 2, 4, 4, odd, p, None) == INVALID
    assert L.sln_mx4_round(None, 0, 2, 4, 4, p, p, None) == INVALID
    assert L.sln_mx4_round(None, 0, 0, 4, 4, None, None, None) == 0
    assert L.sln_mx4_values(p, p, 1, 1, None, 0, None) == INVALID
    assert L.sln_mx4_product(p, p, p, p, 1, 1, 0, None, None, 0, p, 0, None, 0, None) == INVALID
    assert L.sln_mx4_product(p, p, None, p, 1, 1, 8, None, None, 0, p, 0, None, 0, None) == INVALID
    assert L.sln_mx4_product(p, p, p, p, 1, 1, 12544, None, None, 0, p, 0, None, 0, None) == WORKSPACE
    assert L.sln_mx4_product(None, None, None, None, 0, 1, 8, None, None, 0, None, 0, None, 0, None) == 0
    assert L.sln_mx4_rows_product(p, 0, 17, 8, 8, p, p, 1, None, None, 0, p, None, 0, None) == UNSUPPORTED
    assert L.sln_mx4_rows_product(p, 0, 2, 8, 7, p, p, 1, None, None, 0, p, None, 0, None) == INVALID
    assert L.sln_mx4_linear_bwd(p, 0, 3, None, None, p, p, p, p, 2, 4, 8, p, p, p, p, 4096, None) == INVALID
    assert L.sln_mx4_linear_bwd(p, 0, 4, None, None, p, p, None, p, 2, 4, 8, p, None, None, p, 4096, None) == INVALID
    assert L.sln_mx4_linear_bwd(p, 0, 4, None, None, p, p, p, p, 2, 4, 8, p, p, p, odd, 4096, None) == INVALID
    assert L.sln_mx4_linear_bwd(p, 0, 4, None, None, p, p, p, p, 2, 4, 8, p, p, p, p, 16, None) == WORKSPACE
    assert L.sln_mx4_linear_bwd(p, 0, 4, None, None, p, p, p, p, 1 << 22, 4, 8, p, p, p, p, 16, None) == UNSUPPORTED


def test_host_tensors_and_wrong_arguments_are_refused():
    from sln_amodal_amd import ops
    with pytest.raises(RuntimeError):
        ops.mx4_quantize(torch.zeros(2, 32))
    with pytest.raises(TypeError):
        ops.mx4_quantize([1.0])
    with pytest.raises(RuntimeError):
        ops.mx4_linear(torch.zeros(2, 32), torch.zeros(4, 32))
    with pytest.raises(TypeError):
        ops.mx4_linear(None, torch.zeros(4, 32))


def test_kept_codes_do_not_travel_with_a_parameter():
    """Version, address and stream of a weight mean nothing in a copy or another process: what was kept stays behind."""
    import copy
    import io
    import pickle
    from sln_amodal_amd import nn_ops
    kept = nn_ops._Mx4Codes((("version", 1, 2), "codes"))
    assert kept[1] == "codes"
    assert not pickle.loads(pickle.dumps(kept)) and not copy.deepcopy(kept)
    w = torch.nn.Parameter(torch.zeros(2, 3))
    w._sln_mx4_codes = kept
    f = io.BytesIO()
    torch.save(w, f)
    f.seek(0)
    assert not getattr(torch.load(f, weights_only=False), "_sln_mx4_codes", ())


def test_only_products_of_rows_have_a_4bit_form():
    from sln_amodal_amd import nn_ops
    for conv, shape in ((torch.nn.Conv2d(4, 8, 3), (2, 4, 5, 5)), (torch.nn.Conv2d(4, 8, 3, dilation=2), (2, 4, 3, 3)),
                        (torch.nn.Conv2d(4, 8, 3, padding=1), (2, 4, 3, 3)), (torch.nn.Conv2d(4, 8, 1, stride=2), (2, 4, 5, 5)),
                        (torch.nn.Conv2d(4, 8, 1, groups=2), (2, 4, 1, 1))):
        with pytest.raises(RuntimeError, match="no product of rows"):
            nn_ops._mx4_conv(torch.zeros(shape), conv, None, False)


def test_codes_of_a_backward_pass_are_aligned():
    from sln_amodal_amd import _lib
    L = _lib.lib()
    buf = (C.c_char * 8192)()
    p = C.c_void_p((C.addressof(buf) + 255) // 256 * 256)
    odd = C.c_void_p(p.value + 4)
    run = lambda xc, wc: L.sln_mx4_linear_bwd(p, 0, 4, None, None, xc, p, wc, p, 2, 4, 8, p, p, p, p, 4096, None)
    assert run(odd, p) == 1 and run(p, odd) == 1
