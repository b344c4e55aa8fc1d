"""Pools whose rows lie over one another: refused by stores, on the host, before anything is launched (the device pointers here need
not be any)."""

from __future__ import annotations

import pytest

from minisgl_amd.kernel import lib
from test_mx4_cpu import INVALID, pool, rows


# of 10 pages of 16 tokens of 2 heads of 128: 64 bytes of codes a row, 4 of scales
@pytest.mark.parametrize("layout", [
    dict(cp=64), dict(cp=15 * 128 + 64), dict(ct=64), dict(ct=64, ch=128), dict(ct=128, ch=128), dict(ct=64, ch=960), dict(cp=64, ct=64, ch=64),
    dict(cp=64, ct=640, ch=640), dict(cp=128, ct=64, ch=10 * 128),
    dict(sp=4), dict(sp=15 * 8 + 4), dict(st=4), dict(sh=8), dict(st=4, sh=8), dict(st=4, sh=60), dict(sp=4, st=40, sh=40)])
def test_stores_refuse_rows_over_one_another(layout):
    for pools in (dict(kp=pool(**layout)), dict(vp=pool(**layout))):
        rc, message = rows("mla_mx4_store", **pools), lib.load_library().mla_last_error().decode()
        assert rc == INVALID and "over one another" in message, (layout, rc, message)
