"""The slots of a routed batch (moe.cu, route_block), modelled on the CPU: expert counts, a mask of tokens per expert, and from them the
slot of every (token, pick), the slot's token and each token's slots in expert order. All of it counts on a token's picks being k
different experts; what a token without a top k (NaN logits) takes has to keep that."""
import random

import pytest


def scatter(ids, E, GS=2):
    """(slot -> token, token -> slots, tokens of the groups); entries that nothing writes are None."""
    T, K = len(ids), len(ids[0])
    cnt, mask = [0] * E, [0] * E
    for t, row in enumerate(ids):
        for e in row:
            cnt[e] += 1
            mask[e] |= 1 << t
    off = [sum(cnt[:e]) for e in range(E)]
    slot_token, token_slots = [None] * (T * K), [[None] * K for _ in range(T)]
    groups = {(e, j): [None] * min(GS, cnt[e] - GS * j) for e in range(E) for j in range(-(-cnt[e] // GS))}
    for t, row in enumerate(ids):
        for e in row:
            pos = bin(mask[e] & ((1 << t) - 1)).count("1")
            slot_token[off[e] + pos] = t
            groups[e, pos // GS][pos % GS] = t
            token_slots[t][sum(x < e for x in row)] = off[e] + pos
    return slot_token, token_slots, groups


def whole(ids, E):
    slot_token, token_slots, groups = scatter(ids, E)
    flat = [s for row in token_slots for s in row]
    return None not in slot_token and None not in flat and len(set(flat)) == len(flat) and \
        all(None not in g for g in groups.values()) and all(slot_token[s] == t for t, row in enumerate(token_slots) for s in row)


@pytest.mark.parametrize("T", [1, 2, 4, 20, 64])
def test_a_token_without_a_top_k_takes_k_different_experts(T):
    rng = random.Random(T)
    E, K = 16, 4
    for _ in range(20):
        ids = [rng.sample(range(E), K) for _ in range(T)]
        bad = rng.sample(range(T), rng.randint(1, min(T, 3)))
        for t in bad:
            ids[t] = list(range(K))
        assert whole(ids, E)
        for t in bad:
            ids[t] = [0] * K  # one expert k times leaves slots unwritten
        assert not whole(ids, E)
