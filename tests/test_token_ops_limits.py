"""Limits of the token operators' sizes (no GPU): what would leave 32 bits is refused."""
import pytest

from test_token_ops_host import ADDR, attention, refused


@pytest.mark.parametrize("tokens", [2 ** 31 - 255, 2 ** 31 - 129, 2 ** 31 - 64, 2 ** 31 - 1])
@pytest.mark.parametrize("offsets", [0, ADDR])
def test_more_keys_than_a_tile_s_last_place_allows(tokens, offsets):
    refused(attention, "kv_tokens must be", kv_tokens=tokens, documents=1, d_q_offsets=offsets, d_kv_offsets=offsets)
