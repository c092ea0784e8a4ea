"""CPU: what group norm asks for beside its tensors."""
import pytest

from mappedconvolutions_b200 import _lib


@pytest.mark.parametrize("dtype,size", [(_lib.MC_F32, 4), (_lib.MC_F64, 8), (_lib.MC_BF16, 2)])
def test_scratch_grows_with_the_input(dtype, size):
    """Sums of every channel of an image in double (16 bytes), two values of the arithmetic's type for every channel of a tile of at least a
    pixel and for a group; a column of 256 vectors is a tile's least part."""
    L = _lib.lib()
    wide = 8 if size == 8 else 4
    shapes = [(1, 1, 1 << 20), (8, 1, 1 << 20), (64, 1, 65_536), (8, 4096, 8192), (1, 1, (1 << 20) - 1), (1, 7, (1 << 20) - 1), (3, 5, 30_011),
              (2, 9, 2049), (1, 40_962, 256), (64, 10_242, 256), (1000, 4, 24), (5, 1, 7), (1 << 18, 1, 64), (2, 1 << 20, 4)]
    for b, s, c in shapes:
        for layout in (_lib.MC_NHWC, _lib.MC_NCHW):
            for groups in {1, c, max(g for g in range(1, 65) if c % g == 0)}:
                d = _lib.McNormDesc(b, s, c, groups, 0, dtype, layout, 1e-5)
                n = b * s * c
                for phase in (0, 1):
                    got = L.mc_group_norm_workspace_bytes(d, phase)
                    assert 0 < got <= n * (3 * wide + 16 + 2 * wide) + 256 * 16 * 3 * wide + 4096, (b, s, c, groups, layout, phase, got / n)


def test_limits():
    L = _lib.lib()

    def answer(b, s, c, groups, layout):
        d = _lib.McNormDesc(b, s, c, groups, 0, _lib.MC_BF16, layout, 1e-5)
        fits = L.mc_group_norm_workspace_bytes(d, 0) > 0
        assert fits == (L.mc_group_norm_workspace_bytes(d, 1) > 0)
        rc = L.mc_group_norm_fwd(d, *[256] * 6, 16, None)
        assert rc == (-3 if fits else -6)  # the scratch is too small, or the limit is told
        return fits
    for layout in (_lib.MC_NHWC, _lib.MC_NCHW):
        assert answer(1 << 20, 2, 64, 64, layout) and answer(1 << 21, 4, 64, 32, layout) and answer((1 << 25) - 1, 2, 64, 64, layout)
        assert not answer(1 << 25, 2, 64, 64, layout) and not answer(1 << 11, 1, 1 << 20, 1 << 20, layout)
        assert answer((1 << 11) - 1, 1, 1 << 20, 1 << 20, layout)
    assert answer(1, 4096 * 1023, 1 << 20, 1, _lib.MC_NCHW) and not answer(1, 4096 * 1023 + 1, 1 << 20, 1, _lib.MC_NCHW)
