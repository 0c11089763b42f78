"""Copies that a product's kernel has on their way when it gives up land before their buffer is used again or the CTA leaves: read from
the source, since no run brings a late copy about."""

import re

from tests.test_source_order import CSRC, _body


def test_every_wait_that_gives_up_on_copies_lets_them_land():
    text = (CSRC / "product.cu").read_text()
    assert "__nanosleep" in _body(text, "void settle(")
    kernel = _body(text, "\nproduct_kernel(")
    # the producer, behind its ring; the epilogue, whose residual may be on its way: at the accumulator's wait and at its own
    producer, epilogue = kernel[kernel.index("if (warp == kEpiWarps)"):kernel.index("} else if (warp == kEpiWarps + 1)")], kernel[kernel.index("auto ask_residual"):]
    assert re.search(r"if \(dead\) settle\(\);", producer)
    accumulator = _body(epilogue, "if (!have)")
    assert accumulator.index("settle();") < accumulator.index("break;")
    residual = _body(epilogue, "if (!mbar_wait_warp<false>(smem_u32(&s_res[warp][slot])")
    assert "settle();" in residual and "__syncwarp();" in residual[residual.index("settle();"):]
