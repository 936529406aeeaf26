"""Limits of the token operators' sizes (no GPU): what would leave 32 bits is refused."""
import pytest

from test_token_ops_host import ADDR, attention, binding, refused


@pytest.mark.parametrize("tokens", [2 ** 31 - 255, 2 ** 31 - 129, 2 ** 31 - 64, 2 ** 31 - 1])
@pytest.mark.parametrize("offsets", [0, ADDR])
def test_more_keys_than_a_tile_s_last_place_allows(tokens, offsets):
    refused(attention, "kv_tokens must be", kv_tokens=tokens, documents=1, d_q_offsets=offsets, d_kv_offsets=offsets)


@pytest.mark.parametrize("tiles", [0, 1, 3, 4, 5, 8, 9, 30])
def test_no_copy_of_the_attention_s_tiles_is_left_in_flight(tiles):
    """Whichever wait for a stage gives up, every copy that was begun is waited for: through its stage, or
    at the end; those behind the wait that gave up are never begun."""
    needed = 2 * max(0, tiles - 4)  # waits, with four stages of keys and of values
    for waits in range(needed + 1):
        copies = binding().debug_attention_loads(tiles, waits)
        begun = 2 * tiles if waits == needed else 8 + waits
        assert all(c in (2, 3) for c in copies[:begun]) and not any(copies[begun:]), (waits, copies)
        assert copies[:begun].count(3) == min(begun, 8)
