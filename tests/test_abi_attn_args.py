"""Refusals of the operators over the K/V cache (no GPU needed; nothing is enqueued): memory that is written and shared with
another argument, small arrays out of alignment, more query rows than a grid holds."""
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


Q, LSE, TREE = 4 * 24 * 1024, 4 * 24 * 4, 4 * 8
KB = 4 * 64 * 516
TREE_ARGS = {"qn": Q, "k": KV, "v": KV, "pos0": 4, "tree": TREE, "o": Q, "lse": LSE, "ws": 1 << 30}
WEIGHT_ARGS = {"qn": Q, "lse": LSE, "k": KV, "pos0": 4, "tree": TREE, "rows": 8, "acc": ACC}
BLOCK_ARGS = {"qn": Q, "k": KV, "v": KV, "pos0": 4, "idx": 4 * 4 * 64 * 4, "o": Q, "lse": LSE, "ws": 1 << 30}
BOUND_ARGS = {"k": KV, "pos0": 4, "kb": KB}
SELECT_ARGS = {"qn": Q, "kb": KB, "pos0": 4, "idx": 4 * 4 * 64 * 4, "ws": 4 * 4 * 64 * 4}
ACCEPT_ARGS = {"k": KV, "v": KV, "acc": ACC, "pos0": 4, "path": 4 * 4, "n_path": 4}


def tree(ops, **a):
    ops.attn_tree(a["qn"], a["k"], a["v"], a["pos0"], a["tree"], 4, 0.0625, 24, 4, 4096, True, a["o"], WS(1 << 30, a["ws"]), 0, a["lse"])


def weights(ops, **a):
    ops.attn_weights(a["qn"], a["lse"], a["k"], a["pos0"], a["tree"], 4, 0.0625, 24, 4, 4096, True, a["acc"], 0, a["rows"])


def blocks(ops, **a):
    ops.attn_blocks(a["qn"], a["k"], a["v"], a["pos0"], a["idx"], 4, 64, 0.0625, 24, 4, 4096, True, a["o"], WS(1 << 30, a["ws"]), 0, a["lse"])


def bounds(ops, **a):
    ops.kv_block_bounds(a["k"], a["pos0"], 4, 4, 4096, True, a["kb"], 0)


def select(ops, **a):
    ops.attn_select(a["qn"], a["kb"], a["pos0"], 4, 24, 4, 4096, 64, 1, 2, a["idx"], WS(1 << 30, a["ws"]), 0)


def accept(ops, **a):
    ops.kv_accept([a["k"], a["v"]], [a["acc"]], a["pos0"], a["path"], a["n_path"], 4, 4, 4096, True, 0)


@pytest.mark.parametrize("call,args,out,other", [
    (call, args, a, b) for call, args, outs in ((tree, TREE_ARGS, ("o", "lse", "ws")), (weights, WEIGHT_ARGS, ("acc",)),
                                                (blocks, BLOCK_ARGS, ("o", "lse", "ws")), (bounds, BOUND_ARGS, ("kb",)),
                                                (select, SELECT_ARGS, ("idx", "ws")), (accept, ACCEPT_ARGS, ("k", "v", "acc")))
    for a, b in pairs(outs, args) if b != "ws"])
def test_outputs_over_other_arguments_are_refused(q27, call, args, out, other):
    at = {name: (i + 1) * G4 for i, name in enumerate(args)}
    at[out] = at[other] + (args[other] - 1) // 16 * 16
    refused(q27, lambda o: call(o, **at))


def test_evict_pos_refuses_one_place_for_both(q27):
    refused(q27, lambda o: o.kv_evict_pos(G4, G4, 4, 0))


@pytest.mark.parametrize("call,args,name,by", [
    (call, args, name, by) for call, args, names in (
        (tree, TREE_ARGS, {"tree": 4, "lse": 2, "pos0": 1}), (weights, WEIGHT_ARGS, {"tree": 4, "rows": 4, "lse": 2, "acc": 1, "pos0": 2}),
        (blocks, BLOCK_ARGS, {"idx": 2, "lse": 1, "pos0": 2}), (bounds, BOUND_ARGS, {"pos0": 2}), (select, SELECT_ARGS, {"idx": 1, "pos0": 2}),
        (accept, ACCEPT_ARGS, {"acc": 2, "pos0": 1, "path": 2, "n_path": 3})) for name, by in names.items()])
def test_arrays_out_of_alignment_are_refused(q27, call, args, name, by):
    at = {n: (i + 1) * G4 for i, n in enumerate(args)}
    at[name] += by
    refused(q27, lambda o: call(o, **at), needle="alignment")


@pytest.mark.parametrize("name,by", [("acc", 2), ("ao", 1), ("kept", 2), ("pos0", 1)])
def test_evict_arrays_out_of_alignment_are_refused(q27, name, by):
    refused(q27, evict, {name: EVICT[name] * G4 + by}, needle="alignment")
    refused(q27, lambda o: o.kv_evict_pos(G4, 2 * G4 + by, 4, 0), needle="alignment")


@pytest.mark.parametrize("T,nqh,nkvh", [(1, 1 << 24, 1 << 24), (1, 1 << 24, 1), (64, 1 << 18, 4), (64, 1 << 30, 1 << 10), (17, 1 << 29, 1)])
def test_more_query_rows_than_a_grid_holds_are_refused(q27, T, nqh, nkvh):
    a = {n: (i + 1) << 50 for i, n in enumerate(TREE_ARGS)}
    assert q27.ops.attn_tree_ws_bytes(T, nqh, nkvh, 4096) == 0
    refused(q27, lambda o: o.attn_tree(a["qn"], a["k"], a["v"], a["pos0"], None, T, 0.0625, nqh, nkvh, 4096, True, a["o"],
                                       WS(1 << 60, a["ws"]), 0), needle="too many", code=-1)
    refused(q27, lambda o: o.attn_weights(a["qn"], a["lse"], a["k"], a["pos0"], None, T, 0.0625, nqh, nkvh, 4096, True, a["o"], 0),
            needle="too many", code=-1)
