"""Codes of the token mixers' C entries for strides that their kernels' offsets do not cover (placeholders that are never
dereferenced)."""
import pytest

from test_mixers_refusals import OK, P, SHAPE, L, lib, packed  # noqa: F401


@pytest.mark.parametrize("fn", ["step", "prefill"])
def test_values_strides_are_not_negative(lib, fn):              # noqa: F811
    """The scan takes a chunk's values by unsigned 32-bit offsets from its first row."""
    def call(ldv, T=1):
        return getattr(lib, "prism_delta_" + fn)(packed(
            L._ARGS, P, 256, 128, P, 256, 128, P, ldv, 128, P, 4, P, 4, P, 4 * 128 * 128, 2, None, P, 512, 128, P, 1, T, 2, 4,
            128, 128, 1, 1.0, 1e-6, None, 0), None)
    assert call(512, T=0) == OK
    assert call(-512) == SHAPE and call(-512, T=0) == SHAPE
