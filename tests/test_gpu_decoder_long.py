"""The decoder's caches where they fill: what has no room is refused."""
import pytest

from test_gpu_decoder_prompt import PROMPT, _build

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("kv", ["bf16", "e4m3"])
def test_prefill_counts_what_the_cache_holds(dev, kv):
    """Token by token as in one pass: a prompt that does not fit behind the cached tokens is refused,
    one that just fits is not."""
    dec = _build(dev, kv_cache=kv)
    room = dec.cfg.max_seq
    assert room == 64
    for feed in (dec.prefill, dec.prefill_prompt):
        dec.reset()
        feed(PROMPT)
        with pytest.raises(ValueError, match="longer than max_seq"):
            feed(PROMPT[:room - len(PROMPT) + 1])
        assert int(dec.pos.item()) == len(PROMPT)
        feed(PROMPT[:room - len(PROMPT)])
        assert int(dec.pos.item()) == room
