"""What the operators around attention and the experts refuse, before any device work."""
import pytest
import torch


def _rc(name, *args):
    import stade_hip
    L = stade_hip.lib()
    return getattr(L, name)(*args, None), L.stade_hip_last_error().decode()


FAKE = 1 << 20   # (aligned, never read)
A = FAKE
GOOD = {
    "stade_hip_head_rotary": [0, 0, A, 24, A, 24, A, A, A, A, 8, 2, 1, 8, 4, 1, 1, 1e-6, 1.0],
    "stade_hip_head_rotary_b": [0, 0, A, 24, A, 24, A, 24, A, A, A, A, A, A, 8, 2, 1, 8, 4, 1, 1, 1e-6, 1.0, 1],
    "stade_hip_attention": [0, A, 16, A, A, 16, A, 8, A, 8, A, A, 0.5, 8, 2, 1, 4, 4, 1, -1, 0],
    "stade_hip_attention_b": [0, A, 16, A, 16, A, A, 16, A, 16, A, 8, A, 8, A, 8, A, 8, A, A, 0.5, 8, 2, 1, 4, 4, 1, -1, 0, 1],
    "stade_hip_expert_order": [A, A, A, A, 2, 3, 4],
    "stade_hip_expert_take": [0, A, 8, A, 8, A, 8, 2, 4],
    "stade_hip_expert_take_b": [0, A, 8, A, 8, A, 8, 2, 4, 1],
    "stade_hip_expert_join": [0, A, 8, A, 8, A, A, 8, 2, 4, 0],
    "stade_hip_expert_join_b": [0, A, 8, A, 8, A, 8, A, A, A, 8, 2, 4, 1],
    "stade_hip_dropout": [0, A, 8, A, 8, A, 8, A, 0.5, 8, 4],
    "stade_hip_dropout_b": [0, A, 8, A, 8, A, 0.5, 8, 4, 1],
}
INF, NAN, BIG = float("inf"), float("nan"), 1 << 40
BAD = [
    ("stade_hip_head_rotary", 0, 7, -1, "type"), ("stade_hip_head_rotary", 1, 2, -1, "neither"), ("stade_hip_head_rotary", 3, 23, -1, "ldy"),
    ("stade_hip_head_rotary", 5, 23, -1, "ldx"), ("stade_hip_head_rotary", 10, 257, -3, "above"), ("stade_hip_head_rotary", 11, -1, -1, "negative"),
    ("stade_hip_head_rotary", 12, BIG, -3, "above"), ("stade_hip_head_rotary", 13, 7, -1, "odd"), ("stade_hip_head_rotary", 13, 10, -3, "above"),
    ("stade_hip_head_rotary", 14, -1, -1, "negative"), ("stade_hip_head_rotary", 16, 0, -1, "without the norm"), ("stade_hip_head_rotary", 17, -1.0, -1, "eps"),
    ("stade_hip_head_rotary", 17, NAN, -1, "eps"), ("stade_hip_head_rotary", 18, INF, -1, "finite"), ("stade_hip_head_rotary", 4, None, -1, "null"),
    ("stade_hip_head_rotary", 8, None, -1, "null"), ("stade_hip_head_rotary", 9, None, -1, "null"),
    ("stade_hip_head_rotary_b", 0, -1, -1, "type"), ("stade_hip_head_rotary_b", 4, None, -1, "null"), ("stade_hip_head_rotary_b", 2, None, -1, "null"),
    ("stade_hip_head_rotary_b", 7, 20, -1, "ldxb"), ("stade_hip_head_rotary_b", 3, 20, -1, "ldyb"), ("stade_hip_head_rotary_b", 20, 0, -1, "without the norm"),
    ("stade_hip_attention", 0, 3, -1, "type"), ("stade_hip_attention", 2, 15, -1, "ldy"), ("stade_hip_attention", 5, 15, -1, "ldq"),
    ("stade_hip_attention", 7, 7, -1, "ldk"), ("stade_hip_attention", 9, 7, -1, "ldv"), ("stade_hip_attention", 1, None, -1, "null"),
    ("stade_hip_attention", 4, None, -1, "null"), ("stade_hip_attention", 6, None, -1, "null"), ("stade_hip_attention", 10, None, -1, "null"),
    ("stade_hip_attention", 11, None, -1, "null"), ("stade_hip_attention", 12, NAN, -1, "finite"), ("stade_hip_attention", 12, INF, -1, "finite"),
    ("stade_hip_attention", 13, 129, -3, "above"), ("stade_hip_attention", 13, -1, -1, "negative"), ("stade_hip_attention", 14, 3, 0, ""),
    ("stade_hip_attention", 15, 3, -1, "multiple"), ("stade_hip_attention", 15, 0, -1, "multiple"), ("stade_hip_attention", 16, BIG, -3, "above"),
    ("stade_hip_attention", 17, -1, -1, "negative"), ("stade_hip_attention", 18, BIG, -3, "above"), ("stade_hip_attention", 20, 65, -3, "above"),
    ("stade_hip_attention", 20, -1, -1, "negative"),
    ("stade_hip_attention_b", 1, None, -1, "null"), ("stade_hip_attention_b", 3, None, -1, "null"), ("stade_hip_attention_b", 5, None, -1, "null"),
    ("stade_hip_attention_b", 9, 15, -1, "ldqb"), ("stade_hip_attention_b", 13, 7, -1, "ldkb"), ("stade_hip_attention_b", 17, 7, -1, "ldvb"),
    ("stade_hip_attention_b", 2, 15, -1, "ldyb"), ("stade_hip_attention_b", 21, 200, -3, "above"),
    ("stade_hip_expert_order", 0, None, -1, "null"), ("stade_hip_expert_order", 2, None, -1, "null"), ("stade_hip_expert_order", 3, None, -1, "null"),
    ("stade_hip_expert_order", 4, 65, -3, "above"), ("stade_hip_expert_order", 5, 5000, -3, "above"), ("stade_hip_expert_order", 6, 1 << 30, -3, "above"),
    ("stade_hip_expert_take", 0, 9, -1, "type"), ("stade_hip_expert_take", 2, 7, -1, "ldxs"), ("stade_hip_expert_take", 4, 7, -1, "ldx"),
    ("stade_hip_expert_take", 5, None, -1, "null"), ("stade_hip_expert_take", 7, -1, -1, "negative"),
    ("stade_hip_expert_take_b", 2, 7, -1, "ldxsb"), ("stade_hip_expert_take_b", 3, None, -1, "null"), ("stade_hip_expert_take_b", 1, None, -1, "null"),
    ("stade_hip_expert_join", 4, 7, -1, "ldys"), ("stade_hip_expert_join", 1, None, -1, "null"), ("stade_hip_expert_join", 6, None, -1, "null"),
    ("stade_hip_expert_join_b", 3, None, -1, "null"), ("stade_hip_expert_join_b", 1, None, -1, "null"), ("stade_hip_expert_join_b", 6, 7, -1, "ldysb"),
    ("stade_hip_expert_join_b", 9, None, -1, "null"), ("stade_hip_expert_join_b", 12, BIG, -3, "above"),
    ("stade_hip_dropout", 0, 4, -1, "type"), ("stade_hip_dropout", 8, 1.0, -1, "p is not"), ("stade_hip_dropout", 8, -0.1, -1, "p is not"),
    ("stade_hip_dropout", 8, NAN, -1, "p is not"), ("stade_hip_dropout", 8, 0.999999, -1, "p is not"), ("stade_hip_dropout", 7, None, -1, "null"),
    ("stade_hip_dropout", 6, 7, -1, "ldr"), ("stade_hip_dropout", 2, 7, -1, "ldy"), ("stade_hip_dropout", 9, -8, -1, "negative"),
    ("stade_hip_dropout_b", 4, 7, -1, "ldxb"), ("stade_hip_dropout_b", 1, None, -1, "null"), ("stade_hip_dropout_b", 6, 2.0, -1, "p is not"),
]
BAD = [b for b in BAD if b[3]]


@pytest.mark.parametrize("name,at,value,code,text", BAD, ids=[f"{b[0][10:]}-{b[1]}-{b[2]}" for b in BAD])
def test_refused(name, at, value, code, text):
    args = list(GOOD[name])
    args[at] = value
    rc, msg = _rc(name, *args)
    assert rc == code and text in msg and name in msg, (rc, msg)


def test_heads_that_do_not_divide():
    args = list(GOOD["stade_hip_attention"])
    args[14], args[15], args[2], args[5], args[7], args[9] = 3, 2, 24, 24, 16, 16
    rc, msg = _rc("stade_hip_attention", *args)
    assert rc == -1 and "multiple" in msg


def test_rows_past_32_bits():
    args = list(GOOD["stade_hip_attention"])
    args[14], args[15], args[16], args[2], args[5] = 4096, 1, 1 << 20, 8 * 4096, 8 * 4096
    rc, msg = _rc("stade_hip_attention", *args)
    assert rc == -3 and "above" in msg


def test_frequencies_refused():
    import stade_hip
    for bad, text in ((dict(i_r=7), "odd"), (dict(i_r=600), "above"), (dict(i_r=8, base=0.0), "positive"), (dict(i_r=8, factor=-1.0), "positive"),
                      (dict(i_r=8, length=-1.0), "length"), (dict(i_r=8, length=100.0, low=4.0, high=4.0), "low"), (dict(i_r=8, base=NAN), "positive")):
        with pytest.raises(stade_hip.StadeHipError, match=text):
            stade_hip.rotary_freq(**bad)
    with pytest.raises(ValueError, match="negative"):
        stade_hip.rotary_freq(-2)


def test_extents_of_zero_need_no_device():
    assert _rc("stade_hip_head_rotary", 0, 0, None, 24, None, 24, None, None, None, None, 8, 2, 1, 8, 0, 1, 1, 1e-6, 1.0)[0] == 0
    assert _rc("stade_hip_head_rotary_b", 0, 0, None, 24, None, 24, None, 24, None, None, None, None, None, None, 8, 2, 1, 8, 0, 1, 1, 1e-6, 1.0, 0)[0] == 0
    assert _rc("stade_hip_attention", 0, None, 16, None, None, 16, None, 8, None, 8, FAKE, FAKE, 0.5, 8, 2, 1, 0, 4, 1, -1, 0)[0] == 0
    assert _rc("stade_hip_attention_b", 0, None, 16, None, 16, None, None, 16, None, 16, None, 8, None, 8, None, 8, None, 8, FAKE, FAKE, 0.5, 8, 2, 1, 0, 0, 1,
               -1, 0, 0)[0] == 0
    assert _rc("stade_hip_expert_take", 0, None, 8, None, 8, None, 8, 2, 0)[0] == 0
    assert _rc("stade_hip_expert_join", 0, None, 8, None, 8, None, None, 8, 2, 0, 0)[0] == 0
    assert _rc("stade_hip_expert_join_b", 0, None, 8, None, 8, None, 8, None, None, None, 8, 0, 3, 0)[0] == 0
    assert _rc("stade_hip_dropout", 0, None, 8, None, 8, None, 8, None, 0.5, 0, 4)[0] == 0
    assert _rc("stade_hip_dropout_b", 0, None, 8, None, 8, None, 0.5, 8, 0, 1)[0] == 0


def test_python_checks():
    import stade_hip
    x, i = torch.zeros(4, 8), torch.zeros(4, dtype=torch.int64)
    with pytest.raises(ValueError, match="not on a GPU"):
        stade_hip.head_rotary(x, x, None, None, i, x, 8, 1, 0, 8, 4)
    with pytest.raises(ValueError, match="not on a GPU"):
        stade_hip.attention(x, None, x, x, x, i, i, 1.0, 8, 1, 1, 4, 4, 3)
    with pytest.raises(TypeError, match="float32, bfloat16 or float16"):
        stade_hip.dropout(x.double(), x.double(), None, i, 0.5, 8, 4)
    with pytest.raises(TypeError, match="torch tensor"):
        stade_hip.expert_take(x, None, i, 8, 1, 4)
    with pytest.raises(TypeError, match="Int64"):
        stade_hip.expert_join(x, x, None, i, 8.0, 1, 4)
    with pytest.raises(ValueError, match="negative"):
        stade_hip.expert_order(i, i, i, i, 1, -1, 4)
    with pytest.raises(ValueError, match="negative"):
        stade_hip.attention(x, None, x, x, x, i, i, 1.0, 8, 1, 1, 4, 4, 3, window=-1)
