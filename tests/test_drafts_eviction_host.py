"""The refusals of the operators that verify drafts, gather attention weights and evict from the cache: arguments are looked at
before anything is launched, so they are tested without a GPU."""
from types import SimpleNamespace

import pytest
import torch

from qwen_engine_b200 import ops
from qwen_engine_b200.sampling import Sampler, SamplingParams


def _empty(shape, dtype):
    return torch.empty(shape, dtype=dtype)


def _verify_args(**other):
    N, R, V = 5, 2, 11
    a = dict(logits=torch.zeros(N, V), draft_tokens=torch.zeros(N - R, dtype=torch.int32), draft_logits=torch.zeros(N - R, V),
             row_starts=torch.tensor([0, 3, 5], dtype=torch.int32), temperature=torch.ones(R), top_k=torch.zeros(R, dtype=torch.int32),
             uniform=torch.zeros(N), tokens=torch.zeros(N, dtype=torch.int32), counts=torch.zeros(R, dtype=torch.int32), alloc=_empty)
    a.update(other)
    return a


@pytest.mark.parametrize("other", [
    dict(logits=torch.zeros(5, 11, dtype=torch.bfloat16)), dict(logits=torch.zeros(11, 5).T), dict(draft_tokens=torch.zeros(4, dtype=torch.int32)),
    dict(draft_tokens=torch.zeros(3, dtype=torch.int64)), dict(draft_logits=torch.zeros(3, 12)), dict(draft_logits=torch.zeros(3, 11, dtype=torch.float64)),
    dict(row_starts=torch.zeros(2, dtype=torch.int32)), dict(temperature=torch.ones(3)), dict(temperature=torch.ones(2, dtype=torch.float64)),
    dict(top_k=torch.zeros(2)), dict(uniform=torch.zeros(4)), dict(tokens=torch.zeros(4, dtype=torch.int32)), dict(uniform=torch.zeros(10)[::2])])
def test_verify_drafts_refuses(other):
    with pytest.raises(ops.KernelRefused):
        ops.verify_drafts(**_verify_args(**other))


def test_operands_on_the_cpu_are_refused():
    with pytest.raises(ops.ExtensionMissing):
        ops.verify_drafts(**_verify_args())
    with pytest.raises(ops.ExtensionMissing):
        ops.accumulate_attention(**_weights_args())
    with pytest.raises(ops.ExtensionMissing):
        ops.evict_tokens(**_evict_args())


def _weights_args(**other):
    R, Hq, Hkv, D, P, slots, cap = 2, 4, 2, 16, 8, 3, 40
    ctx = SimpleNamespace(num_reqs=R, cu_q=torch.tensor([0, 2, 3], dtype=torch.int32), ctx_lens=torch.tensor([5, 9], dtype=torch.int32),
                          slot_ids=torch.tensor([0, 2], dtype=torch.int32), positions=torch.zeros(3, dtype=torch.int32),
                          q_lens_host=[2, 1], ctx_lens_host=[5, 9])
    a = dict(qkv=torch.zeros(3, (Hq + 2 * Hkv) * D), kv_pages=torch.zeros(6, 2, Hkv, P, D), block_tables=torch.zeros(R, 2, dtype=torch.int32),
             ctx=ctx, weights=torch.zeros(slots, Hkv, cap), out=torch.zeros(slots, Hkv, cap), scale=0.25, window=0, num_heads=Hq,
             num_kv_heads=Hkv, head_dim=D, alloc=_empty)
    a.update(other)
    return a


_ONE = torch.zeros(3 * 2 * 40 + 4)


@pytest.mark.parametrize("other", [
    dict(qkv=torch.zeros(3, 128, dtype=torch.bfloat16)), dict(qkv=torch.zeros(128, 3).T), dict(qkv=torch.zeros(3, 60)), dict(num_heads=5),
    dict(kv_pages=torch.zeros(6, 2, 3, 8, 16)), dict(kv_pages=torch.zeros(6, 2, 8, 16)), dict(kv_pages=torch.zeros(6, 2, 2, 8, 32)[..., ::2]),
    dict(block_tables=torch.zeros(2, 2, dtype=torch.int64)), dict(block_tables=torch.zeros(3, 2, dtype=torch.int32)),
    dict(block_tables=torch.zeros(2, 1, dtype=torch.int32)),                         # 10 tokens in one block of 8
    dict(weights=torch.zeros(3, 2, 9), out=torch.zeros(3, 2, 9)),                    # ... and in 9 places
    dict(weights=torch.zeros(3, 2, 40, dtype=torch.float64)), dict(out=torch.zeros(3, 2, 41)),
    dict(weights=_ONE[:240].view(3, 2, 40), out=_ONE[4:].view(3, 2, 40)),            # they overlap
    dict(positions=torch.zeros(3, 2, 40)), dict(counted=torch.zeros(3, dtype=torch.int32)), dict(counted=torch.zeros(2)),
    dict(slopes=torch.zeros(2)), dict(sinks=torch.zeros(4, dtype=torch.float64)), dict(scale=0.0), dict(softcap=-1.0)])
def test_accumulate_attention_refuses(other):
    with pytest.raises(ops.KernelRefused):
        ops.accumulate_attention(**_weights_args(**other))


def _evict_args(**other):
    S, R, Hkv, D, P, slots, cap = 2, 2, 2, 16, 8, 3, 16
    a = dict(cache=torch.zeros(S, 6, 2, Hkv, P, D), block_tables=torch.zeros(R, 2, dtype=torch.int32), slot_ids=torch.tensor([0, 2], dtype=torch.int32),
             lens=torch.tensor([12, 16], dtype=torch.int32), weights=torch.zeros(S, slots, Hkv, cap),
             positions=torch.zeros(S, slots, Hkv, cap, dtype=torch.int32), weights_out=torch.zeros(S, slots, Hkv, cap),
             positions_out=torch.zeros(S, slots, Hkv, cap, dtype=torch.int32), keep=8, first=1, recent=3, alloc=_empty)
    a.update(other)
    return a


@pytest.mark.parametrize("other", [
    dict(cache=torch.zeros(6, 2, 2, 8, 16)), dict(cache=torch.zeros(2, 6, 2, 2, 16, 8).transpose(4, 5)),
    dict(cache=torch.zeros(2, 6, 2, 2, 8, 15, dtype=torch.uint8)), dict(block_tables=torch.zeros(3, 2, dtype=torch.int32)),
    dict(slot_ids=torch.zeros(3, dtype=torch.int32)), dict(lens=torch.zeros(2)), dict(weights=torch.zeros(1, 3, 2, 16)),
    dict(weights=torch.zeros(2, 3, 2, 16, dtype=torch.bfloat16)), dict(positions=torch.zeros(2, 3, 2, 17, dtype=torch.int32)),
    dict(weights_out=torch.zeros(2, 3, 2, 17)), dict(positions_out=torch.zeros(2, 3, 2, 16)), dict(keep=0), dict(first=-1), dict(recent=-1),
    dict(keep=8, first=5, recent=4)])
def test_evict_tokens_refuses(other):
    with pytest.raises(ops.KernelRefused):
        ops.evict_tokens(**_evict_args(**other))


def test_the_sampler_refuses_lists_that_do_not_fit():
    s = Sampler("cpu")
    p = [SamplingParams(temperature=1.0)] * 2
    for drafts, uniforms, rows in [([[1]], [[0.1, 0.2]], 2), ([[1], []], [[0.1, 0.2], []], 3), ([[1], []], [[0.1, 0.2], [0.3]], 4)]:
        with pytest.raises(ValueError):
            s.verify(torch.zeros(rows, 9), p, drafts, uniforms)


def test_parts_of_rows():
    """Tiles that give every SM four CTAs are not cut; fewer are cut into as many parts as do, of a tile of the other side at least."""
    assert ops._attention_weights_parts(600, 32) == 1 and ops._attention_weights_parts(592, 32) == 1
    assert ops._attention_weights_parts(100, 32) == 6 and ops._attention_weights_parts(8, 5) == 5 and ops._attention_weights_parts(1, 0) == 1
    assert ops._attention_weights_parts(1, 1 << 13) == ops.ATTENTION_WEIGHTS_MAX_PARTS


def test_where_a_few_rows_scores_go():
    """Short contexts of few requests: a cluster's shared memory, parts that hold every key; else scratch memory, parts of 512 to 2 048 keys."""
    for rows in (1, 2, 16, 17, 32):
        for span in (1, 31, 32, 33, 1000, 4096, 4097, 100000):
            for requests in (1, 2, 3, 64):
                ctas, part = ops.attention_weights_cluster(rows, 8, 128, requests, span)
                assert part % 32 == 0
                if ctas:
                    assert ctas == 8 and ctas * part >= span and requests <= 2 and span <= 4096
                else:
                    assert 512 <= part <= 2048 and (requests > 2 or span > 4096 or ops._cluster_smem(rows, 128, -(-span // 256) * 32) > 110 * 1024)
    for units in (1, 7, 64, 1000):
        for tiles in (1, 3, 4, 100):
            parts = ops.attention_weights_tc_parts(units, tiles)
            assert 1 <= parts <= max(1, -(-tiles // 4)) and (parts == 1 or (parts - 1) * units < 4 * 148)


def test_the_entry_points_take_what_the_fronts_give():
    """The types by which ctypes converts the arguments, against the entry points' declarations."""
    import os
    import re
    folder = os.path.join(os.path.dirname(os.path.abspath(ops.__file__)), "..", "csrc")
    source = "".join(open(os.path.join(folder, f)).read() for f in sorted(os.listdir(folder)) if f.endswith(".cu"))
    for name, types in ops._SIGNATURES.items():
        declared = re.search(r'extern "C" int ' + name + r"\(([^)]*)\)", source).group(1).split(",")
        kinds = [ops._P if "*" in d or "cudaStream_t" in d else ops._L if d.strip().startswith("long ") else ops._F if d.strip().startswith("float ") else ops._I
                 for d in declared]
        assert kinds == types, name


@pytest.mark.parametrize("name,value", [
    ("cu_q", torch.tensor([0, 2, 3])), ("cu_q", torch.tensor([0, 2], dtype=torch.int32)), ("cu_q", torch.zeros(6, dtype=torch.int32)[::2]),
    ("ctx_lens", torch.tensor([5, 9])), ("ctx_lens", torch.tensor([5], dtype=torch.int32)), ("slot_ids", torch.tensor([0, 2])),
    ("slot_ids", torch.tensor([0], dtype=torch.int32)), ("positions", torch.zeros(3, dtype=torch.int64)), ("positions", torch.zeros(2, dtype=torch.int32)),
    ("q_lens_host", [2]), ("ctx_lens_host", [5, 9, 1]), ("q_lens_host", [2, 2])])
def test_accumulate_attention_refuses_a_context_that_does_not_fit(name, value):
    """What the kernels read of the step's context: int32, a number for every request (cu_q one more) and for every row."""
    args = _weights_args()
    setattr(args["ctx"], name, value)
    with pytest.raises(ops.KernelRefused, match="accumulate_attention"):
        ops.accumulate_attention(**args)


def test_logits_that_are_no_rows_are_refused():
    with pytest.raises(ops.KernelRefused):
        ops.verify_drafts(**_verify_args(logits=torch.zeros(55)))


def test_kernels_are_configured_for_every_device_they_run_on():
    """A kernel's attributes hold for one device: no launcher of these operators sets them once a process."""
    import os
    import re
    folder = os.path.join(os.path.dirname(os.path.abspath(ops.__file__)), "..", "csrc")
    for name in ("verify.cu", "evict.cu", "attention_weights.cu", "attention_weights_few.cu", "attention_weights_tc.cu"):
        source = open(os.path.join(folder, name)).read()
        assert "static bool" not in source, name
        for at in re.finditer("cudaFuncSetAttribute", source):
            assert "qe_once_a_device(" in source[max(0, at.start() - 120):at.start()], name


def _manager(num_pages=12):
    from qwen_engine_b200.cache import CacheManager, PagedKVSpec
    return CacheManager([PagedKVSpec(2, 8)] * 2 + [PagedKVSpec(1, 8)], 4, num_pages, 6, torch.float32, "cpu")


def _opened(cm, name, tokens):
    rc = cm.open(name, tokens, len(tokens))
    cm.append(rc, tokens[rc.num_tokens:])
    cm.commit(rc)
    return rc


def test_private_pages_are_not_found_by_their_tokens():
    """Pages within which entries are moved: a request that is opened later with the same tokens must not get them, neither those that were full
    when they became private nor those that become full afterwards."""
    prompt = list(range(30, 42))
    cm = _manager()
    a = _opened(cm, "a", prompt[:10])
    cm.make_private(a, 0)
    assert cm.open("b", prompt, 12).shared_tokens == 0
    cm.close(cm.live["b"])
    cm.append(a, prompt[10:])
    cm.commit(a)
    assert cm.open("c", prompt, 12).shared_tokens == 0 and cm.page_copies_by_group() == {}
    cm.check_invariants()
    # ... nor when they have been given back
    cm.close(a)
    cm.close(cm.live["c"])
    assert cm.open("d", prompt, 12).shared_tokens == 0
    cm.check_invariants()


def test_pages_that_others_hold_are_copied_before_they_become_private():
    prompt = list(range(30, 42))
    cm = _manager()
    a = _opened(cm, "a", prompt)
    b = _opened(cm, "b", prompt[:9])
    assert b.shared_tokens == 8
    held = list(b.tables[0])
    cm.make_private(a, 0)
    assert b.tables[0] == held and a.tables[0][:2] != held[:2] and not set(a.tables[0]) & set(held)
    assert cm.page_copies_by_group() == {0: [held[0], a.tables[0][0], held[1], a.tables[0][1]]}
    assert a.tables[1][:2] == b.tables[1][:2]             # (the other group's are as they were)
    cm.check_invariants()
    # b's stay findable; a's third page was found through no copy
    c = cm.open("c", prompt, 12)
    assert c.shared_tokens == 8 and c.tables[0] == held[:2]
    cm.check_invariants()
    for rc in (a, b, c):
        cm.close(rc)
    cm.check_invariants()


def test_pages_do_not_become_private_by_halves():
    from qwen_engine_b200.cache import OutOfPages
    prompt = list(range(30, 42))
    cm = _manager(num_pages=5)
    a, b = _opened(cm, "a", prompt), _opened(cm, "b", prompt[:9])
    tables = [list(a.tables[0]), list(b.tables[0])]
    with pytest.raises(OutOfPages):
        cm.make_private(a, 0)
    assert [a.tables[0], b.tables[0]] == tables and cm.page_copies_by_group() == {} and not a.private
    assert cm.open("c", prompt, 12).shared_tokens == 11   # (all of it is found; the last page is copied)
    cm.check_invariants()


def test_parts_of_prompts_give_every_sm_a_unit():
    """As many parts as give every SM one, and no more; four tiles of the other side a part at least."""
    for units in (1, 2, 7, 64, 74, 147, 148, 149, 1000):
        for tiles in (1, 3, 4, 5, 100, 1000):
            parts = ops.attention_weights_tc_parts(units, tiles)
            assert 1 <= parts <= min(max(1, -(-tiles // 4)), ops.ATTENTION_WEIGHTS_MAX_PARTS) and (parts == 1 or (parts - 1) * units < 148)
            assert parts * units >= 148 or parts in (-(-tiles // 4), ops.ATTENTION_WEIGHTS_MAX_PARTS)
