"""What the gated block's operators (libsdfnn.so) refuse, copy or look at before they launch anything: no GPU needed."""
import pytest
import torch

from sdfstudio_amd import _nn

P = 4096  # a non-null, 16-byte aligned address nobody reads


def apart(rows, dim, stride, t):
    """rows x dim with `stride` elements between rows (memory that is never touched)."""
    return torch.empty((rows - 1) * stride + dim, dtype=t).as_strided((rows, dim), (stride, 1))


def test_rows_far_apart_are_copied_for_the_products():
    for t, es in ((torch.bfloat16, 2), (torch.float32, 4), (torch.int8, 1)):
        near, far = (1 << 23) // es - 16, (1 << 23) // es
        for stride, copied in ((near, False), (far, True), (far + 16, True)):
            x = apart(3, 32, stride, t)
            x.copy_(torch.arange(96).view(3, 32) % 50)
            kept, at, rows, ld = _nn.rows_of(x, align=True)
            assert rows == 3 and (ld == 32) == copied and (at == x.data_ptr()) == (not copied)
            assert torch.equal(kept, x)
            assert _nn.rows_of(x)[3] == stride  # the norms walk any stride


def test_c_abi_refuses_rows_far_apart_before_it_launches():
    """Also where operands would be copied first (hidden widths that are no multiple of 8)."""
    lib = _nn.load()

    def refused(rc):
        assert rc == -1 and "8 MiB" in _nn.last_error(), (rc, _nn.last_error())

    far16, far8, big = 1 << 22, 1 << 23, 1 << 40
    refused(lib.sdfnn_int8_linear(P, far8, P, P, 64, P, None, 1, 40, 16, 64, P, P, big, None))
    refused(lib.sdfnn_int8_linear(P, 64, P, P, far8, P, None, 1, 40, 16, 64, P, P, big, None))
    refused(lib.sdfnn_int8_gated_linear(P, 64, P, P, 64, P, P, far8, P, 0, 1, 40, 16, 64, P, P, big, None))
    for hidden in (72, 75):
        refused(lib.sdfnn_gated_forward(P, far16, P, P, P, 1, 0, 40, 64, hidden, 64, None, P, P, big, None))
        for rows in (4, 40):
            refused(lib.sdfnn_gated_backward(P, far16, P, P, P, P, P, 64, 1, rows, 64, hidden, 64, P, P, P, P, P, big, None))
            refused(lib.sdfnn_gated_backward(P, 64, P, P, P, P, P, far16, 1, rows, 64, hidden, 64, P, P, P, P, P, big, None))
