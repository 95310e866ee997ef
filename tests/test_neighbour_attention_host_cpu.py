"""What the operators of attention over neighbours do on the host: checks at the entry points, and tables that are made once."""

import ctypes


from lunaequivariance_b200 import _native


def test_wide_cotangents_are_checked():
    """The forms for cotangents in float: refused as their counterparts are, and where 16-bit types are not aligned to 16 bytes."""
    lib = _native.library()
    some, odd = ctypes.c_void_p(16), ctypes.c_void_p(20)
    table = _native.RowTable(2, 4, 0, 0, 16)

    def backward(dtype, alpha=some, g=some, heads=1):
        return lib.luna_graph_softmax_bwd_wide(dtype, ctypes.byref(table), alpha, g, None, None, None, heads, 0, None, 0, None)

    def second(dtype, alpha=some, halpha=some, g=None):
        return lib.luna_graph_softmax_dbl_bwd_wide(dtype, ctypes.byref(table), alpha, g, None, None, None, halpha, None, 1, 0, None, 0, None)

    for dtype in (_native.LUNA_BF16, _native.LUNA_F16):
        assert backward(dtype, g=odd) == backward(dtype, alpha=odd) == _native.LUNA_ERR_MISALIGNED
        assert second(dtype, g=some, halpha=odd) == _native.LUNA_ERR_MISALIGNED
    for dtype in range(4):
        # an output, an operand, a head too few
        assert backward(dtype) == backward(dtype, g=None) == backward(dtype, heads=0) == _native.LUNA_ERR_INVALID_ARGUMENT
        assert second(dtype) == second(dtype, alpha=None, g=some) == _native.LUNA_ERR_INVALID_ARGUMENT
    assert backward(9) == second(9) == _native.LUNA_ERR_INVALID_ARGUMENT
    assert backward(_native.LUNA_F32, g=ctypes.c_void_p(18)) == _native.LUNA_ERR_MISALIGNED
