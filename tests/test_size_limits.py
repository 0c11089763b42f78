"""Sizes at the end of 32 bits: what the kernels count past the end of is refused before any launch."""

import ctypes

from flashrnn_b200 import _lib

END = 2 ** 31


def product_plan(rows, outputs, inputs):
    return _lib.load().frnn_b200_product_plan(rows, outputs, inputs, ctypes.byref(_lib.ProductPlan()))


def test_inputs_of_a_product():
    """Its kernel of few rows goes through the inputs in strides of up to 512: the last stride ends within 32 bits."""
    assert product_plan(1, 8, END - 512) == 0
    for inputs in (END - 504, END - 256, END - 8):
        assert inputs - 1 + 512 >= END and product_plan(1, 8, inputs) == -2


def test_channels_of_the_recurrence():
    """The sum of db rounds the gates' columns up to blocks of 32: that ends within 32 bits too."""
    def plan(function, nd):
        return _lib.load().frnn_b200_linear_plan(_lib.LINEAR_CELLS[function], 2, 1, 1, nd, ctypes.byref(_lib.LinearPlan()))

    for function, gates in (("leaky", 2), ("lstm", 4)):
        assert plan(function, (END - 32) // gates) == 0
        for columns in (END - 28, END - 4):
            assert columns + 31 >= END and plan(function, columns // gates) == -2
