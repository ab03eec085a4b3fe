"""Factors that Float32, in which the kernels take them, does not hold are refused before any device work."""
import pytest

from test_attention_refusals import GOOD, _rc

AT = {"stade_hip_head_rotary": 18, "stade_hip_head_rotary_b": 22, "stade_hip_attention": 12, "stade_hip_attention_b": 20}
TOKENS = {"stade_hip_head_rotary": 14, "stade_hip_head_rotary_b": 18, "stade_hip_attention": 16, "stade_hip_attention_b": 24}


@pytest.mark.parametrize("s", [1e39, -1e39, 3.5e38, 1e300, -1.7e308])
@pytest.mark.parametrize("name", AT)
def test_factor(name, s):
    args = list(GOOD[name])
    args[AT[name]] = s
    rc, msg = _rc(name, *args)
    assert rc == -1 and "s is not finite" in msg and name in msg, (rc, msg)


@pytest.mark.parametrize("eps", [1e39, 1e300, float("inf")])
@pytest.mark.parametrize("name", ["stade_hip_head_rotary", "stade_hip_head_rotary_b"])
def test_eps(name, eps):
    args = list(GOOD[name])
    args[AT[name] - 1] = eps
    rc, msg = _rc(name, *args)
    assert rc == -1 and "eps" in msg and name in msg, (rc, msg)


@pytest.mark.parametrize("name", AT)
def test_the_largest_is_taken(name):
    """(no tokens, and accumulated: nothing is launched)"""
    args = list(GOOD[name])
    args[AT[name]], args[TOKENS[name]] = -3.4028234e38, 0
    assert _rc(name, *args)[0] == 0
