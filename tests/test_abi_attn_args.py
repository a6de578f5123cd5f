"""Refusals of the operators over the K/V cache that depend on two arguments at once: memory that is written and shared with
another argument (no GPU needed; nothing is enqueued)."""
import pytest

from test_abi_attn import WS

G4 = 1 << 32  # the buffers of a call lie 4 GiB apart
KV, ACC = 4 * 4096 * 272, 4 * 4096 * 4  # bytes of a cache and of a weight array


def refused(q27, call, *args, needle="overlap", code=-4):
    with pytest.raises(q27.Q27Error) as ei:
        call(q27.ops, *args)
    assert ei.value.code == code and needle in str(ei.value)


EVICT = {"k": 1, "v": 2, "acc": 3, "ko": 4, "vo": 5, "ao": 6, "kept": 7, "ws": 8, "pos0": 9}


def evict(o, at):
    a = {k: n * G4 for k, n in EVICT.items()} | at
    o.kv_evict(a["k"], a["v"], a["acc"], a["pos0"], 64, 4, 16, a["ko"], a["vo"], a["ao"], 128 if a["ao"] != a["acc"] else 4096,
               a["kept"], 4, 4096, True, WS(1 << 30, a["ws"]), 0)


SIZES = {"k": KV, "v": KV, "acc": ACC, "ko": 4 * 128 * 272, "vo": 4 * 128 * 272, "ao": 4 * 128 * 4, "kept": 4 * 64 * 4, "pos0": 4}


def pairs(outs, others):
    return [(a, b) for a in outs for b in others if a != b]


@pytest.mark.parametrize("out,other", pairs(["ko", "vo", "ao", "kept", "ws"], SIZES))
def test_evict_refuses_outputs_over_other_arguments(q27, out, other):
    refused(q27, evict, {out: EVICT[other] * G4 + (SIZES[other] - 1) // 16 * 16})  # its last 16 bytes


@pytest.mark.parametrize("out,other", pairs(["kept", "ws"], ["k", "v", "acc", "kept", "pos0"]))
def test_evict_in_place_refuses_lists_and_workspaces_over_the_caches(q27, out, other):
    refused(q27, evict, {"ko": G4, "vo": 2 * G4, "ao": 3 * G4, out: EVICT[other] * G4 + (SIZES[other] - 1) // 16 * 16})


@pytest.mark.parametrize("at", [{"acc": G4 + 1024, "ao": G4 + 1024}, {"acc": 2 * G4, "ao": 2 * G4}])
def test_evict_in_place_refuses_weights_in_a_cache(q27, at):
    refused(q27, evict, {"ko": G4, "vo": 2 * G4} | at)
