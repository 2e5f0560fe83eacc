"""CPU-only: what the matrix operators refuse at the ends of their range, before any GPU is touched."""
import ctypes as C

import pytest

pytest.importorskip("torch")
from test_products_host import NMFk, ORTHO, _cf, _last  # noqa: F401,E402


@pytest.mark.parametrize("c", [(1000.0, -1000.0, 1e-20), (1000.0, -1000.0, -1e-300), (200.0, -201.0, 1e-17), (-500.0, 500.0, 3e-18), (1000.0, -1000.0, 0.0), (0.0, 500.0, -500.0)])
def test_orthogonalize_sees_every_peak_of_the_coefficients(NMFk, c):
    """t (a + b t^2 + c t^4) peaks inside (0, 1) at more than 64, whatever the size of c"""
    keep, at = _cf(*c)
    # (too small a workspace: nothing is launched even if the coefficients pass)
    assert NMFk.lib().nmfk_orthogonalize(*{**ORTHO, "steps": 1, "cf": at, "wb": 16}.values()) == 1
    assert "grow beyond 64" in _last(NMFk.lib())


@pytest.mark.parametrize("c", [(1.5, -0.5, 0.0), (1.875, -1.25, 0.375), (3.4445, -4.7750, 2.0315), (1.5, -0.5, 1e-20), (1.5, -0.5, -1e-20), (0.0, 0.0, 0.0), (0.0, 0.0, 60.0), (64.0, 0.0, 0.0)])
def test_orthogonalize_takes_coefficients_that_stay_bounded(NMFk, c):
    keep, at = _cf(*c)
    assert NMFk.lib().nmfk_orthogonalize(*{**ORTHO, "steps": 1, "cf": at, "wb": 16}.values()) == 1
    assert "workspace" in _last(NMFk.lib())
