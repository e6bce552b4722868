"""The split of a short text in a long cache (CPU): at most 2048 chunks, and messages that say so."""
import ctypes

import pytest

import rapier_amd as rmi

AT = [ctypes.c_void_p(1 << (24 + i)) for i in range(16)]


def decode(max_ctx, nsub):
    far = [ctypes.c_void_p(i << 42) for i in range(1, 6)]
    rmi._call("rmi_gqa_tree_decode", AT[0], 1, far[0], 1, far[1], AT[1], None, None, 0, far[2], 4096, None, 0, far[3], 16, 4, 256, 1, max_ctx,
              nsub, 0.0625, None)


@pytest.mark.parametrize("max_ctx", [262145, 1 << 20, 1 << 30])
@pytest.mark.parametrize("text,ntok", [(1, 1), (4096, 1), (4096, 64), (100, 999)])
def test_a_short_texts_split_in_a_long_cache(max_ctx, text, ntok):
    split = rmi.gqa_tree_nsub(text, 16, 4, 256, ntok)
    flag, nsub = split & rmi.TREE_SHORT, split & (rmi.TREE_SHORT - 1)
    least = -(-max_ctx // 262144)
    for n in (nsub, least - 1):
        if 0 < n < least:
            with pytest.raises(ValueError, match="2048 chunks"):
                rmi.gqa_tree_workspace_bytes(max_ctx, 16, 4, 256, ntok, n + flag)
            with pytest.raises(ValueError, match="2048 chunks"):
                decode(max_ctx, n + flag)
    assert rmi.gqa_tree_workspace_bytes(max_ctx, 16, 4, 256, ntok, max(nsub, least) + flag) > 0
    assert rmi.gqa_tree_workspace_bytes(262144, 16, 4, 256, ntok, nsub + flag) > 0
