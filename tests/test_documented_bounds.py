"""CPU checks that the workspace sizes stay within what the header says of them."""
import re

from conftest import ROOT
from onereel_amd import _lib as L


def test_partial_gradients_of_the_attention():
    header = (ROOT / 'include' / 'onereel_hip.h').read_text()
    bound = 10 ** 6 * int(re.search(r'gradients of the tiles that a call of up to 64 segments may split \(up to (\d+) MB\)',
                                    re.sub(r'\s*\n \*\s*', ' ', header)).group(1))
    size, most = L.lib().or_varlen_bwd_workspace_size, 0
    for H in range(1, 257):
        for D in (64, 128):
            for n in (700, 4000, 32 * 256 * 128 // H):
                for n_seg in (1, 64):
                    # without two floats a query row and head, and the tile tables (16 and 32 bytes an item)
                    rest = 8 * H * n + 48 * (3 * n // 128 + 3 * n_seg + 2000) + 2048
                    most = max(most, size(n_seg, n, n, n, n, H, D) - rest)
    assert 0.95 * bound < most <= bound
