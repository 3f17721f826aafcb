"""Outputs whose own heads share memory are refused, on the host; every other stride is taken up to the launch."""

import ctypes
import itertools

import pytest

import ekv_hip
from test_append_refusals import appending, rotation

KINDS = {"ekv_rotate_heads": rotation, "ekv_append_tokens": appending}


def outcome(name, **over):
    """'shared', or what else the call is refused for (a table's stride is looked at behind the outputs, so that no case
    gets to a device)."""
    with pytest.raises(ValueError) as refused:
        ekv_hip.call(name, ctypes.addressof(KINDS[name](**over)), 0)
    return "shared" if "share memory" in str(refused.value) else str(refused.value)


@pytest.mark.parametrize("token,head", [(0, 64), (512, 0), (0, 0), (504, 64), (64, 64), (512, 56), (64, 128), (128, 256), (-504, 64)])
def test_append_refuses_queries_that_overlap(token, head):
    assert outcome("ekv_append_tokens", q_out_stride_token=token, q_out_stride_head=head, table_stride=3) == "shared"


@pytest.mark.parametrize("which,heads", [("q_out", 8), ("k_out", 2)])
@pytest.mark.parametrize("token,head", [(0, 64), (64, 0), (0, 0), (56, 64), (64, 64)])
def test_rotation_refuses_outputs_that_overlap(which, heads, token, head):
    assert outcome("ekv_rotate_heads", **{f"{which}_stride_token": token, f"{which}_stride_head": head}) == "shared"


# (128, 192): 3 tokens of 8 heads at different multiples of 64
@pytest.mark.parametrize("token,head", [(512, 64), (64, 192), (128, 192), (1024, 128), (520, 64), (-512, 64), (512, -64),
                                        (1 << 40, 1 << 20)])
def test_outputs_that_lie_apart_are_taken(token, head):
    assert "stride" in outcome("ekv_append_tokens", q_out_stride_token=token, q_out_stride_head=head, table_stride=3)


def test_one_token_or_one_head_of_any_stride():
    assert "stride" in outcome("ekv_append_tokens", tokens=1, rows=1, q_out_stride_token=0, table_stride=3)
    assert "stride" in outcome("ekv_append_tokens", q_heads=1, q_out_stride_head=0, table_stride=3)
    assert "stride" in outcome("ekv_append_tokens", q_heads=0, query=0, q_out=0, q_out_stride_token=0, q_out_stride_head=0, table_stride=3)


def test_every_small_pair_of_strides():
    """Against the rows themselves, of 16 elements."""
    for tokens, heads in ((2, 2), (3, 4), (5, 2), (4, 7)):
        for token, head in itertools.product(range(0, 160, 8), repeat=2):
            starts = sorted(t * token + h * head for t in range(tokens) for h in range(heads))
            shared = any(b - a < 16 for a, b in zip(starts, starts[1:]))
            got = outcome("ekv_append_tokens", tokens=tokens, rows=tokens, q_heads=heads, head_dim=16, pairs=8, table_stride=3,
                          q_out_stride_token=token, q_out_stride_head=head)
            assert (got == "shared") == shared, (tokens, heads, token, head)
