"""What the language-model operators refuse, before any device work."""
import ctypes

import pytest
import torch


def _lib():
    import stade_hip
    return stade_hip.lib()


FAKE = 1 << 20   # (aligned, never read)


def _rc(name, *args):
    L = _lib()
    return getattr(L, name)(*args, None), L.stade_hip_last_error().decode()


GOOD = {
    "stade_hip_embed": [0, 0, FAKE, 8, FAKE, 8, FAKE, 1.0, 8, 4, 2],
    "stade_hip_embed_b": [0, 0, FAKE, 8, FAKE, 8, FAKE, 1.0, 8, 4, 2, 1],
    "stade_hip_token_order": [FAKE, FAKE, FAKE, 4, 2],
    "stade_hip_tape8_store": [0, FAKE, 8, FAKE, FAKE, 8, 2],
    "stade_hip_tape8_load": [0, FAKE, FAKE, FAKE, 8, 8, 2],
    "stade_hip_layernorm": [0, 0, FAKE, 8, FAKE, 8, FAKE, FAKE, FAKE, FAKE, None, None, 8, 2, 1e-5],
    "stade_hip_layernorm_b": [0, 0, FAKE, 8, FAKE, 8, None, None, FAKE, 8, FAKE, FAKE, FAKE, FAKE, FAKE, 8, 2, 1],
    "stade_hip_expert_mul": [0, FAKE, 8, FAKE, 8, FAKE, FAKE, 8, 8, 2, 1, 0],
    "stade_hip_expert_mul_b": [0, 0, FAKE, 8, FAKE, 8, None, None, FAKE, 8, FAKE, FAKE, FAKE, 8, 8, 2, 1, 1],
}

BAD = [
    ("stade_hip_embed", 0, 7, -1, "type"), ("stade_hip_embed", 1, -1, -1, "type"), ("stade_hip_embed", 8, -1, -1, "negative"),
    ("stade_hip_embed", 8, 1 << 40, -3, "above"), ("stade_hip_embed", 10, 1 << 40, -3, "above"), ("stade_hip_embed", 3, 7, -1, "ldy"),
    ("stade_hip_embed", 5, 0, -1, "ldw"), ("stade_hip_embed", 2, None, -1, "null"), ("stade_hip_embed", 6, None, -1, "null"),
    ("stade_hip_embed_b", 1, 3, -1, "type"), ("stade_hip_embed_b", 9, -1, -1, "negative"), ("stade_hip_embed_b", 3, 1, -1, "ldyb"),
    ("stade_hip_embed_b", 4, None, -1, "null"), ("stade_hip_token_order", 2, None, -1, "null"), ("stade_hip_token_order", 3, -1, -1, "negative"),
    ("stade_hip_tape8_store", 0, 9, -1, "type"), ("stade_hip_tape8_store", 3, FAKE + 4, -1, "aligned"), ("stade_hip_tape8_store", 2, 7, -1, "ldx"),
    ("stade_hip_tape8_load", 3, None, -1, "null"), ("stade_hip_tape8_load", 6, -2, -1, "negative"),
    ("stade_hip_layernorm", 1, 2, -1, "neither"), ("stade_hip_layernorm", 10, FAKE, -1, "together"), ("stade_hip_layernorm", 14, -1.0, -1, "eps"),
    ("stade_hip_layernorm", 14, float("nan"), -1, "eps"), ("stade_hip_layernorm", 4, None, -1, "null"), ("stade_hip_layernorm", 12, 1 << 30, -3, "above"),
    ("stade_hip_layernorm_b", 4, None, -1, "one of x"), ("stade_hip_layernorm_b", 6, FAKE, -1, "one of x"),
    ("stade_hip_layernorm_b", 13, None, -1, "null"), ("stade_hip_layernorm_b", 9, 7, -1, "ldxb"),
    ("stade_hip_expert_mul", 0, 5, -1, "type"), ("stade_hip_expert_mul", 6, None, -1, "null"), ("stade_hip_expert_mul", 10, 5000, -3, "above"),
    ("stade_hip_expert_mul", 2, 7, -1, "ldy"), ("stade_hip_expert_mul", 5, None, -1, "null"),
    ("stade_hip_expert_mul_b", 1, 1, -1, "neither"), ("stade_hip_expert_mul_b", 4, None, -1, "one of x"),
    ("stade_hip_expert_mul_b", 6, FAKE, -1, "one of x"), ("stade_hip_expert_mul_b", 10, None, -1, "null"),
]


@pytest.mark.parametrize("name,at,value,code,text", BAD, ids=[f"{b[0][10:]}-{b[1]}-{b[2]}" for b in BAD])
def test_refused(name, at, value, code, text):
    args = list(GOOD[name])
    args[at] = value
    rc, msg = _rc(name, *args)
    assert rc == code and text in msg and name in msg, (rc, msg)


def test_extents_of_zero_need_no_device():
    assert _rc("stade_hip_embed", 0, 0, None, 8, None, 8, None, 1.0, 8, 4, 0)[0] == 0
    assert _rc("stade_hip_embed_b", 0, 0, None, 8, None, 8, None, 1.0, 8, 4, 0, 1)[0] == -1       # wb is missing
    assert _rc("stade_hip_tape8_store", 0, None, 0, None, None, 0, 5)[0] == 0
    assert _rc("stade_hip_layernorm", 0, 0, None, 0, None, 0, None, None, None, None, None, None, 0, 3, 1e-5)[0] == 0
    assert _rc("stade_hip_expert_mul", 0, None, 8, None, 8, None, FAKE, 8, 8, 0, 1, 0)[0] == 0


def test_python_checks():
    import stade_hip
    x = torch.zeros(4, 8)
    with pytest.raises(ValueError, match="not on a GPU"):
        stade_hip.layernorm(x, x, None, None, None, None, 8, 4)
    with pytest.raises(ValueError, match="not on a GPU"):
        stade_hip.embed(x, x, torch.zeros(4, dtype=torch.int64), 1.0, 8, 4, 4)
    with pytest.raises(TypeError, match="float32, bfloat16 or float16"):
        stade_hip.tape8_store(x.double(), None, None, 8, 4)
    with pytest.raises(TypeError, match="Int64"):
        stade_hip.expert_mul(x, x, x, x, 8.0, 8, 4, 1)
    with pytest.raises(ValueError, match="negative"):
        stade_hip.token_order(x, x, x, -1, 4)
    with pytest.raises(ValueError, match="one of x and tape"):
        stade_hip.layernorm_b(x, None, x, None, None, None, x, x, 8, 4)
    with pytest.raises(TypeError, match="torch tensor"):
        stade_hip.embed([1.0], x, None, 1.0, 8, 4, 4)
    assert stade_hip.tape8_lengths(0, 5) == (0, 0)
    with pytest.raises(stade_hip.StadeHipError, match="negative"):
        stade_hip.tape8_lengths(-1, 5)
