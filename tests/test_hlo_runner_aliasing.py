"""Custom calls that write over an operand (output_to_operand_aliasing) in the module runner: a value that is read
afterwards keeps what it held."""
import numpy as np
import pytest
import torch

from xla_amd import hlo, hlo_runner

MODULE = """HloModule m, entry_computation_layout={()->()}
ENTRY main {
  moves = s32[1,2] parameter(0)
  a = s8[4,16] parameter(1)
  b = f32[4,3] parameter(2)
  first = (s8[4,16], f32[4,3]) custom-call(moves, a, b), custom_call_target="xla_amd.kv_cache_copy_pages", output_to_operand_aliasing={{0}: (1, {}), {1}: (2, {})}, api_version=API_VERSION_TYPED_FFI
  a1 = s8[4,16] get-tuple-element(first), index=0
  more = s32[1,2] parameter(3)
  second = s8[4,16] custom-call(more, a1), custom_call_target="xla_amd.kv_cache_copy_pages", output_to_operand_aliasing={{}: (1, {})}, api_version=API_VERSION_TYPED_FFI
  %s
}
"""
ROOTS = {"what was written last": ("ROOT r = (s8[4,16]) tuple(second)", (False, False, False)),
         "an input": ("ROOT r = (s8[4,16], s8[4,16]) tuple(second, a)", (True, False, False)),
         "the other input": ("b1 = f32[4,3] get-tuple-element(first), index=1\n  ROOT r = (s8[4,16], f32[4,3], f32[4,3]) tuple(second, b1, b)",
                             (False, True, False)),
         "what lay between": ("ROOT r = (s8[4,16], s8[4,16]) tuple(second, a1)", (False, False, True)),
         "the first call's tuple": ("ROOT r = ((s8[4,16], f32[4,3]), s8[4,16]) tuple(first, second)", (False, False, True))}


@pytest.mark.parametrize("root", ROOTS)
def test_what_is_still_read(root):
    text, want = ROOTS[root]
    entry = next(c for c in hlo.to_json(MODULE % text)["computations"] if c["entry"])["instructions"]
    at = {i["name"]: k for k, i in enumerate(entry)}
    moves, a, b = object(), object(), object()
    assert hlo_runner._aliased(entry[at["first"]]) == {0: 1, 1: 2} and hlo_runner._aliased(entry[at["second"]]) == {0: 1}
    env = {"moves": moves, "a": a, "b": b}
    got = [hlo_runner.still_read(entry, at["first"], env, [moves, a, b], i) for i in (1, 2)]
    a1 = object()
    env.update(first=[a1, b], a1=a1, more=object())
    got.append(hlo_runner.still_read(entry, at["second"], env, [env["more"], a1], 1))
    assert tuple(got) == want
    # one buffer for two operands: each is read by the other
    assert hlo_runner.still_read(entry, at["first"], env, [moves, a, a], 1)


def test_a_tuple_in_a_tuple():
    text = MODULE.replace("  second =", "  nest = ((s8[4,16], f32[4,3]), s32[1,2]) tuple(first, more)\n  second =")
    for root, want in (("inner = (s8[4,16], f32[4,3]) get-tuple-element(nest), index=0\n  ROOT r = (s8[4,16], (s8[4,16], f32[4,3])) tuple(second, inner)", True),
                       ("m = s32[1,2] get-tuple-element(nest), index=1\n  ROOT r = (s8[4,16], s32[1,2]) tuple(second, m)", False)):
        entry = next(c for c in hlo.to_json(text % root)["computations"] if c["entry"])["instructions"]
        at = [i["name"] for i in entry].index("second")
        a1, b1, more = object(), object(), object()
        env = {"first": [a1, b1], "a1": a1, "more": more, "nest": [[a1, b1], more]}
        assert hlo_runner.still_read(entry, at, env, [more, a1], 1) == want


@pytest.mark.gpu
@pytest.mark.parametrize("root", ROOTS)
def test_a_module_that_reads_what_a_call_has_written_over(root):
    rng = np.random.default_rng(3)
    a = torch.from_numpy(rng.integers(-99, 99, (4, 16)).astype(np.int8)).cuda()
    b = torch.from_numpy(rng.standard_normal((4, 3)).astype(np.float32)).cuda()
    moves = [torch.tensor([m], dtype=torch.int32, device="cuda") for m in ([0, 2], [1, 3])]
    want = {"a": a.clone(), "b": b.clone(), "a1": a.clone(), "b1": b.clone()}
    want["a1"][2], want["b1"][2] = a[0], b[0]
    want["second"] = want["a1"].clone()
    want["second"][3] = want["a1"][1]
    want["first"] = [want["a1"], want["b1"]]
    text = ROOTS[root][0]
    got, rewrites, _ = hlo_runner.compile_and_run(MODULE % text, [moves[0], a, b, moves[1]])
    assert not rewrites

    def same(g, w):
        return all(same(x, y) for x, y in zip(g, w)) if isinstance(w, list) else torch.equal(g, w)
    names = text[text.index("tuple(") + 6:-1].split(", ")
    for g, n in zip(got, names):
        assert same(g, want[n]), n
