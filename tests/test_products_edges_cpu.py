"""Calls of the products over 16-bit weights through the binding, without a GPU: what is decided before a device is touched."""
import pytest

from __graft_entry__ import load_package

pkg = load_package()
P = 1 << 20      # an aligned address that no refused call reads


@pytest.fixture
def bare():
    """The binding without a handle: a call that passes every check of its arguments ends at "null handle"."""
    m = pkg.MoE.__new__(pkg.MoE)
    m._h = None
    return m


def refusal(call):
    with pytest.raises(pkg.MlxsError) as ei:
        call()
    return ei.value


def test_a_limit_without_an_activation_says_nothing(bare):
    """A layer keeps one limit for its gate-and-up and its down product."""
    for act in (pkg.GROUPED_SWIGLU, pkg.GROUPED_PLAIN):
        e = refusal(lambda: bare.grouped(P, P, P, P, 16, 4, 256, 128, act=act, act_limit=10.0))
        assert e.rc == pkg.E_ARG and "null handle" in e.msg
    e = refusal(lambda: bare.grouped(P, P, P, P, 16, 4, 256, 128, act=pkg.GROUPED_SWIGLU, act_limit=-1.0))
    assert e.rc == pkg.E_CONFIG and "act_limit" in e.msg
