"""Calls of the Python operators on 4-bit matrices that the interface allows, without a device."""
import ctypes as C

import pytest

from rns8_amd import abi
from test_mx4_abi import NoContext, P, Tensor, lib  # noqa: F401


class Bytes(Tensor):
    def __init__(self, size):
        super().__init__((size,), "uint8")

    def element_size(self):
        return 1


@pytest.mark.parametrize("more", [{}, dict(w_t=Tensor((2 * 2176,), "uint8")), dict(x=Tensor((4, 32))),
                                  dict(x=Tensor((4, 32)), w_t=Tensor((2 * 2176,), "uint8"))])
def test_operands_that_the_wanted_gradients_do_not_read(lib, more):  # noqa: F811
    """A program that wants dbias alone may pass the other operands of the layer all the same."""
    from rns8_amd import operators as ops

    call = ops.LinearMx4Backward(NoContext(), dy=Tensor((4, 8)), dbias=Tensor((8,)), workspace=Bytes(1 << 16), **more)
    args = call.args
    assert (args.m, args.n, args.dbias, args.dx, args.dw) == (4, 8, P, None, None)
    need = C.c_uint64()
    assert lib.rns8_mi355x_linear_mx4_backward_workspace(C.byref(args), C.byref(need)) == abi.SUCCESS
