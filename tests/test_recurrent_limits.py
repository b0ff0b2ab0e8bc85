"""What causal_conv, selective_scan and their steps refuse or plan at the limits of their sizes, without a GPU."""
import ctypes as C

import pytest
import torch

from lasp_b200 import _cabi, causal_conv, causal_conv_step, selective_scan, selective_scan_step
from tests.test_recurrent_calls import P, conv_args, scan_args, tokens

MOST = 2147480000   # channels, and tokens: what lies a tile beyond is still a 32-bit number


def test_channels_that_32_bits_do_not_hold_with_a_tile_more():
    lib = _cabi.load()
    assert lib.lasp_b200_conv_forward(C.byref(conv_args(channels=MOST + 1)), None) == -9
    assert lib.lasp_b200_conv_backward(C.byref(conv_args(channels=MOST + 1, ws_bytes=1 << 60)), None) == -9
    for f in (lib.lasp_b200_scan_forward, lib.lasp_b200_scan_backward):
        assert f(C.byref(scan_args(channels=MOST + 1)), None) == -9
    step = dict(channels=MOST + 1, dtype=_cabi.BF16, slot_count=2, y=tokens(), state=P)
    assert lib.lasp_b200_conv_step(C.byref(_cabi.ConvStepArgs(rows=2, width=4, x=tokens(), weight=P, **step)), None) == -9
    assert lib.lasp_b200_scan_step(C.byref(_cabi.ScanStepArgs(rows=2, states=1, groups=1, A=P, **{k: tokens() for k in ("u", "dt", "B", "C")}, **step)), None) == -9
    wide = lambda *s: torch.zeros(()).expand(*s)   # noqa: E731
    n = MOST + 1
    with pytest.raises(ValueError):
        causal_conv(wide(1, 1, n), wide(n, 4))
    with pytest.raises(ValueError):
        causal_conv_step(wide(1, 3, n), wide(1, n), wide(n, 4))
    with pytest.raises(ValueError):
        selective_scan(wide(1, 1, n), wide(1, 1, n), wide(n, 1), wide(1, 1, 1), wide(1, 1, 1))
    with pytest.raises(ValueError):
        selective_scan_step(wide(1, n, 1), wide(1, n), wide(1, n), wide(n, 1), wide(1, 1), wide(1, 1))


@pytest.mark.parametrize("dtype,states,two_blocks", [(_cabi.BF16, 16, True), (_cabi.F32, 16, False), (_cabi.BF16, 32, True), (_cabi.F32, 32, True),
                                                     (_cabi.F16, 64, False), (_cabi.F32, 64, False)])
def test_two_segments_backward_only_where_an_sm_has_two_blocks(dtype, states, two_blocks):
    """A pass of 99 to 148 blocks on 148 SMs could be cut in two.  Where an SM's shared memory holds one block that takes as long as whole rows,
    and the first pass; three segments (75 to 98 blocks) pay.  Cut or not is seen from the workspace."""
    lanes = 4 if states <= 16 else 8 if states <= 32 else 16

    def bytes_more(tiles):
        c, n = tiles * 128 // lanes, 16384
        need = _cabi.load().lasp_b200_scan_workspace_bytes(C.byref(scan_args(tokens=n, channels=c, states=states, dtype=dtype)))
        return need - 4 * (tiles * n * 8 * lanes + tiles * 512 + 2 * c)   # of a row that is whole

    for tiles in (99, 128, 148):
        assert (bytes_more(tiles) > 0) == two_blocks, tiles
    assert all(bytes_more(tiles) > 0 for tiles in (98, 75, 64, 20, 1)) and bytes_more(198) == 0
    assert bytes_more(149) > 0 and bytes_more(197) > 0   # (three, where some SMs would have twice as much as others)
