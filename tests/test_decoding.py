"""Decoding operators on the host: refusals, masks, the handle -- CPU only."""

from __future__ import annotations

import ctypes

import pytest
import torch

import piper_kernels as pk
from oracle import decoding as oracle
from piper_kernels import _native


def _cache(pages=3, heads=2, page=16, d=64, **kw) -> pk.QuantizedKVCache:
    return pk.QuantizedKVCache.allocate(pages, heads, page, d, device="cpu", **kw)


def _batch(b=2, width=2):
    return torch.zeros((b, width), dtype=torch.int32), torch.zeros(b, dtype=torch.int32)


def test_a_new_cache_stands_for_zeros() -> None:
    c = _cache()
    assert (c.kv_heads, c.page_size, c.head_dim) == (2, 16, 64)
    assert not c.key_codes.any() and bool((c.value_scales == 1).all())


@pytest.mark.parametrize(("change", "match"), [
    (dict(page=24), "page_size"), (dict(page=512), "page_size"), (dict(d=96), "head dimensions"),
    (dict(pages=0), "at least one page"), (dict(key_mean=torch.zeros(2, 63)), "key_mean"),
    (dict(key_mean=torch.zeros(2, 64, dtype=torch.float16)), "float32"),
])
def test_cache_refuses(change, match) -> None:
    with pytest.raises(ValueError, match=match):
        _cache(**change)


def test_cache_refuses_buffers_that_do_not_belong_together() -> None:
    c = _cache()
    with pytest.raises(ValueError, match="value_codes must have shape"):
        pk.QuantizedKVCache(c.key_codes, c.key_scales, c.value_codes[:2], c.value_scales)
    with pytest.raises(ValueError, match="key_scales must use float32"):
        pk.QuantizedKVCache(c.key_codes, c.key_scales.half(), c.value_codes, c.value_scales)
    with pytest.raises(ValueError, match="contiguous"):
        pk.QuantizedKVCache(c.key_codes, c.key_scales, torch.zeros(3, 16, 2, 64, dtype=torch.int8).transpose(1, 2),
                            c.value_scales)


@pytest.mark.parametrize(("change", "match"), [
    (dict(key=torch.zeros(2, 2, 3, 64)), "float16 or bfloat16"),
    (dict(key=torch.zeros(2, 2, 64).half()), "shape"),
    (dict(key=torch.zeros(2, 3, 3, 64).half()), "key must have shape"),
    (dict(value=torch.zeros(2, 2, 4, 64).half()), "value must have shape"),
    (dict(value=torch.zeros(2, 2, 3, 64).bfloat16()), "value must use float16"),
    (dict(value=torch.zeros(2, 2, 64, 3).half().transpose(2, 3)), "last dimension must be contiguous"),
    (dict(key=torch.zeros(2, 2, 0, 64).half(), value=torch.zeros(2, 2, 0, 64).half()), "empty"),
    (dict(block_table=torch.zeros((2, 2), dtype=torch.int64)), "block_table must use int32"),
    (dict(block_table=torch.zeros((3, 2), dtype=torch.int32)), "block_table must have shape"),
    (dict(block_table=torch.zeros((2, 0), dtype=torch.int32)), "at least one column"),
    (dict(lengths=torch.zeros(3, dtype=torch.int32)), "lengths"),
    (dict(counts=torch.zeros(2, dtype=torch.int64)), "counts must use int32"),
    (dict(lengths=torch.zeros(2, dtype=torch.int32, device="meta")), "must be on cpu"),
])
def test_write_refuses(change, match) -> None:
    table, lengths = _batch()
    args = dict(key=torch.zeros(2, 2, 3, 64).half(), value=torch.zeros(2, 2, 3, 64).half(), block_table=table,
                lengths=lengths, counts=None) | change
    with pytest.raises(ValueError, match=match):
        pk.write_kv_cache(_cache(), **args)


@pytest.mark.parametrize(("change", "match"), [
    (dict(query=torch.zeros(2, 4, 3, 64)), "float16 or bfloat16"),
    (dict(query=torch.zeros(2, 4, 64).half()), "shape"),
    (dict(query=torch.zeros(2, 4, 3, 128).half()), "query must have shape"),
    (dict(query=torch.zeros(2, 3, 3, 64).half()), "multiple of the cache's 2 KV heads"),
    (dict(query=torch.zeros(2, 4, 65, 64).half()), "1 to 64 nodes"),
    (dict(query=torch.zeros(2, 4, 0, 64).half()), "1 to 64 nodes"),
    (dict(query=torch.zeros(0, 4, 3, 64).half()), "empty batch"),
    (dict(tree_mask=torch.zeros((2, 3), dtype=torch.int32)), "tree_mask must use int64"),
    (dict(tree_mask=torch.zeros((2, 4), dtype=torch.int64)), "tree_mask must have shape"),
    (dict(scale=0.0), "scale must be finite and positive"),
    (dict(scale=float("nan")), "scale must be finite and positive"),
])
def test_attention_refuses(change, match) -> None:
    table, lengths = _batch()
    args = dict(query=torch.zeros(2, 4, 3, 64).half(), block_table=table, lengths=lengths) | change
    with pytest.raises(ValueError, match=match):
        pk.tree_attention(args.pop("query"), _cache(), **args)


@pytest.mark.parametrize(("change", "match"), [
    (dict(target_probs=torch.zeros(2, 5)), "target_probs must have shape"),
    (dict(target_probs=torch.zeros(2, 3, 5).half()), "target_probs must use float32"),
    (dict(draft_probs=torch.zeros(2, 3, 6)), "draft_probs must have shape"),
    (dict(draft_probs=torch.zeros(2, 5, 3).transpose(1, 2)), "contiguous"),
    (dict(tokens=torch.zeros((2, 3), dtype=torch.int32)), "tokens must use int64"),
    (dict(parents=torch.zeros((2, 3), dtype=torch.int64)), "parents must use int32"),
    (dict(uniform=torch.zeros(2, 4)), "uniform must have shape"),
    (dict(noise=torch.zeros(2, 4)), "noise must have shape"),
])
def test_verify_refuses(change, match) -> None:
    args = dict(target_probs=torch.zeros(2, 3, 5), draft_probs=torch.zeros(2, 3, 5),
                tokens=torch.zeros((2, 3), dtype=torch.int64), parents=torch.zeros((2, 3), dtype=torch.int32),
                uniform=torch.zeros(2, 3), noise=torch.zeros(2, 5)) | change
    with pytest.raises(ValueError, match=match):
        pk.verify_draft_tree(**args)


def test_keep_and_read_refuse() -> None:
    table, lengths = _batch()
    path, counts = torch.zeros((2, 3), dtype=torch.int32), torch.ones(2, dtype=torch.int32)
    with pytest.raises(ValueError, match="path must use int32"):
        pk.keep_draft_path(_cache(), table, lengths, path.long(), counts)
    with pytest.raises(ValueError, match="1 to 64 nodes"):
        pk.keep_draft_path(_cache(), table, lengths, torch.zeros((2, 65), dtype=torch.int32), counts)
    with pytest.raises(ValueError, match="counts must have shape"):
        pk.keep_draft_path(_cache(), table, lengths, path, counts[:1])
    with pytest.raises(ValueError, match="tokens must be positive"):
        pk.read_kv_cache(_cache(), table, lengths, 0)
    with pytest.raises(ValueError, match="float16 or bfloat16"):
        pk.read_kv_cache(_cache(), table, lengths, 1, dtype=torch.float32)


def test_there_is_no_cpu_fallback_and_no_autograd() -> None:
    table, lengths = _batch()
    x = torch.zeros(2, 2, 3, 64).half()
    for call in (
        lambda: pk.write_kv_cache(_cache(), x, x, table, lengths),
        lambda: pk.read_kv_cache(_cache(), table, lengths, 2),
        lambda: pk.keep_draft_path(_cache(), table, lengths, torch.zeros((2, 3), dtype=torch.int32), lengths),
        lambda: pk.tree_attention(x, _cache(), table, lengths),
        lambda: pk.verify_draft_tree(torch.zeros(1, 1, 5), torch.zeros(1, 1, 5), torch.zeros((1, 1), dtype=torch.int64),
                                     torch.zeros((1, 1), dtype=torch.int32), torch.zeros(1, 1), torch.zeros(1, 5)),
    ):
        with pytest.raises(RuntimeError, match="no CPU or generic-GPU fallback"):
            call()
    with pytest.raises(RuntimeError, match="autograd"):
        pk.tree_attention(x.clone().requires_grad_(), _cache(), table, lengths)


def test_entry_points_check_arguments_on_the_host() -> None:
    lib = _native.library()
    good = dict(key_codes=256, key_scales=256, value_codes=256, value_scales=256, key_mean=None, block_table=256,
                lengths=256, pages=2, table_stride=1, kv_heads=1, page_size=16, head_dim=64, batch=1, table_width=1)
    strides = _native._STRIDES(1, 1, 1)

    def refused(call, *args, match, **change):
        cache = _native.KVCache(**(good | change))
        assert call(ctypes.byref(cache), *args) == _native.ERR_INVALID_ARGUMENT
        assert match in _native.last_error()

    read = (256, 256, 0, 1, None, None)
    refused(lib.piper_b200_kv_cache_read, *read, match="head_dim", head_dim=32)
    refused(lib.piper_b200_kv_cache_read, *read, match="page_size", page_size=48)
    refused(lib.piper_b200_kv_cache_read, *read, match="NULL", lengths=None)
    refused(lib.piper_b200_kv_cache_read, *read, match="positive", table_width=0)
    refused(lib.piper_b200_kv_cache_read, *read, match="2^31", pages=1 << 40)
    refused(lib.piper_b200_kv_cache_read, *read, match="16-byte", key_codes=8)
    refused(lib.piper_b200_kv_cache_read, 256, 256, 0, 0, None, None, match="tokens")
    refused(lib.piper_b200_kv_cache_write, None, strides, 256, strides, 0, 1, None, None, match="NULL")
    refused(lib.piper_b200_kv_cache_write, 256, strides, 256, strides, 5, 1, None, None, match="dtype")
    refused(lib.piper_b200_kv_cache_keep, 256, 1, 65, 256, None, match="nodes")
    tree = (256, strides, 256, 0)
    refused(lib.piper_b200_tree_attention, *tree, 1, 0, None, 0, 0.1, None, 0, None, match="nodes")
    refused(lib.piper_b200_tree_attention, *tree, 3, 1, None, 0, 0.1, None, 0, None, match="multiple", kv_heads=2)
    refused(lib.piper_b200_tree_attention, *tree, 1, 1, None, 0, -1.0, None, 0, None, match="scale")
    two = _native._STRIDES2(1, 1)
    for vocab, nodes, match in ((0, 1, "vocab"), (5, 65, "nodes")):
        assert lib.piper_b200_verify_draft_tree(256, two, 256, two, 256, 1, 256, 1, 256, 1, 256, 1, 1, nodes, vocab,
                                                256, 256, 256, None) == _native.ERR_INVALID_ARGUMENT
        assert match in _native.last_error()


def test_tree_mask_from_parents() -> None:
    parents = torch.tensor([[-1, 0, 0, 1, 3, 2], [-1, 0, 1, 2, 3, 4]], dtype=torch.int32)
    mask = pk.tree_mask_from_parents(parents)
    assert mask.tolist() == [[1, 0b11, 0b101, 0b1011, 0b11011, 0b100101], [1, 3, 7, 15, 31, 63]]
    assert pk.tree_mask_from_parents(parents[0]).tolist() == mask[0].tolist()
    chain = pk.tree_mask_from_parents(torch.arange(-1, 63))
    assert chain[63].item() == -1 and chain[62].item() == (1 << 63) - 1
    with pytest.raises(ValueError, match="1 to 64"):
        pk.tree_mask_from_parents(torch.zeros(65, dtype=torch.int32))
    with pytest.raises(ValueError, match="int32 or int64"):
        pk.tree_mask_from_parents(torch.zeros(3))


def test_oracle_verification_follows_the_target_distribution() -> None:
    # One root with two drafted children: the first emitted token's frequencies
    # over many seeds are the target's, whatever the draft.  Each count is
    # binomial; five standard deviations (plus one) bound it.
    g = torch.Generator().manual_seed(7)
    vocab, tries = 4, 4000
    target = torch.softmax(torch.randn((1, 1, vocab), generator=g), -1)
    draft = torch.softmax(torch.randn((1, 1, vocab), generator=g), -1)
    tokens = torch.zeros((tries, 3), dtype=torch.int64)
    tokens[:, 1:] = torch.multinomial(draft[0, 0], 2 * tries, replacement=True, generator=g).view(tries, 2)
    parents = torch.tensor([[-1, 0, 0]], dtype=torch.int32).expand(tries, 3)
    path, count, following = oracle.verify(
        target.expand(tries, 3, vocab), draft.expand(tries, 3, vocab), tokens, parents,
        torch.rand((tries, 3), generator=g), torch.empty((tries, vocab)).exponential_(generator=g))
    first = torch.where(count > 1, tokens.gather(1, path[:, 1:2].long().clamp(min=0))[:, 0], following)
    for x in range(vocab):
        p = float(target[0, 0, x])
        assert abs(int((first == x).sum()) - tries * p) <= 5 * (tries * p * (1 - p)) ** 0.5 + 1


def test_the_binding_passes_on_what_it_does_not_take() -> None:
    # None: the checks that explain come next.  (On CPU tensors that is always so.)
    binding = _native.binding()
    table, lengths = _batch()
    x = torch.zeros(2, 2, 3, 64).half()
    buffers = _cache().buffers
    assert binding.attend(buffers, x, table, lengths, None, None) is None
    assert binding.attend(None, x, table, lengths, None, None) is None
    assert binding.attend(buffers, "query", table, None, 3, 1) is None
    assert binding.attend() is None
    assert binding.write(buffers, x, None, table, lengths, None) is None
    assert binding.read(buffers, table, lengths, None, 1 << 80, True) is None
    assert binding.read((1, 2, 3, 4, 5), table, lengths, None, 1, True) is None
    assert binding.keep(buffers, table, lengths, x, lengths) is None
    assert binding.verify(x, x, x, x, x, x) is None


def test_missing_binding_fails_loudly(monkeypatch: pytest.MonkeyPatch, tmp_path) -> None:
    monkeypatch.setattr(_native, "_binding", None)
    monkeypatch.setattr(_native, "BINDING_PATH", tmp_path / "absent.so")
    with pytest.raises(_native.NativeLibraryMissing, match="build"):
        _native.binding()


def _operators_of(graph_module) -> list[str]:
    return [str(n.target) for n in graph_module.graph.nodes if str(n.target).startswith("piper_kernels.")]


def test_traced_calls_record_the_registered_operators(monkeypatch: pytest.MonkeyPatch) -> None:
    # (Fake tensors need no GPU; only the device's check would ask for one.)
    from torch._subclasses.fake_tensor import FakeTensorMode
    from torch.fx.experimental.proxy_tensor import make_fx

    from piper_kernels.decoding import attention, cache, verification

    for module in (attention, cache, verification):
        monkeypatch.setattr(module, "require_device", lambda *_: None)

    def step(c, x, table, lengths, probs, tokens, parents, path, uniform, noise):
        pk.write_kv_cache(c, x, x, table, lengths)
        out = pk.tree_attention(x, c, table, lengths) + 1
        found = pk.verify_draft_tree(probs, probs, tokens, parents, uniform, noise)
        pk.keep_draft_path(c, table, lengths, path, lengths)
        return out, *found, *pk.read_kv_cache(c, table, lengths, 2)

    with FakeTensorMode():
        kw = dict(device="cuda")
        handle = pk.QuantizedKVCache.allocate(3, 2, 16, 64, device="cuda")
        ints = torch.zeros((2, 3), dtype=torch.int32, **kw)
        args = (torch.zeros((2, 2, 3, 64), dtype=torch.float16, **kw), ints, ints[:, 0].contiguous(),
                torch.zeros((2, 3, 5), **kw), torch.zeros((2, 3), dtype=torch.int64, **kw), ints, ints,
                torch.zeros((2, 3), **kw), torch.zeros((2, 5), **kw))
        shapes = [tuple(x.shape) for x in step(handle, *args)]
        traced = make_fx(lambda *a: step(handle, *a))(*args)
    assert shapes == [(2, 2, 3, 64), (2, 3), (2,), (2,), (2, 2, 2, 64), (2, 2, 2, 64)]
    assert [name.split(".")[1] for name in _operators_of(traced)] == [
        "write_kv_cache", "tree_attention", "verify_draft_tree", "keep_draft_path", "read_kv_cache"]


def test_the_workspace_function_refuses_what_the_call_refuses() -> None:
    # In a process of its own: an integer division by zero would end it.
    import subprocess
    import sys
    from pathlib import Path

    code = """
import sys
sys.path.insert(0, sys.argv[1])
from piper_kernels.decoding.attention import workspace_bytes
good = dict(batch=1, heads=4, kv_heads=4, nodes=1, head_dim=64, positions=4096)
assert workspace_bytes(**good) > 0 and workspace_bytes(**(good | dict(positions=64))) == 0
for match, change in [("multiple", dict(heads=2)), ("multiple", dict(heads=6)), ("multiple", dict(heads=0)),
                      ("nodes", dict(nodes=65)), ("nodes", dict(nodes=0)), ("positive", dict(kv_heads=0)),
                      ("positive", dict(positions=-1)), ("65535", dict(batch=1 << 40)), ("2^39", dict(positions=1 << 62)),
                      ("head_dim", dict(head_dim=96))]:
    try:
        workspace_bytes(**(good | change))
    except ValueError as refused:
        assert match in str(refused), (change, refused)
    else:
        raise AssertionError(change)
"""
    package = Path(pk.__file__).resolve().parents[1]
    done = subprocess.run([sys.executable, "-c", code, str(package)], capture_output=True, text=True, timeout=300)
    assert done.returncode == 0, (done.returncode, done.stderr)


@pytest.mark.parametrize("scale", [1e-46, 1e-39, 2.4e38, 1e39, 5e-324])
def test_scales_that_fp32_does_not_hold_are_refused(scale) -> None:
    table, lengths = _batch()
    with pytest.raises(ValueError, match="scale"):
        pk.tree_attention(torch.zeros(2, 4, 3, 64).half(), _cache(), table, lengths, scale=scale)
    lib = _native.library()
    cache = _native.KVCache(key_codes=256, key_scales=256, value_codes=256, value_scales=256, key_mean=None,
                            block_table=256, lengths=256, pages=2, table_stride=1, kv_heads=1, page_size=16,
                            head_dim=64, batch=1, table_width=1)
    assert lib.piper_b200_tree_attention(ctypes.byref(cache), 256, _native._STRIDES(1, 1, 1), 256, 0, 1, 1, None, 0,
                                         scale, None, 0, None) == _native.ERR_INVALID_ARGUMENT
    assert "scale" in _native.last_error()


def test_a_handle_cannot_be_changed_and_notices_changed_buffers() -> None:
    c = _cache(pages=4)
    for name, value in (("buffers", c.buffers[:4] + (None,)), ("page_size", 32), ("pages", 9), ("kv_heads", 1),
                        ("head_dim", 128), ("device", torch.device("cuda"))):
        with pytest.raises(AttributeError):
            setattr(c, name, value)
    table, lengths = _batch()
    x, ints = torch.zeros(2, 2, 3, 64).half(), torch.zeros((2, 3), dtype=torch.int32)
    calls = (lambda c: pk.write_kv_cache(c, x, x, table, lengths), lambda c: pk.read_kv_cache(c, table, lengths, 2),
             lambda c: pk.keep_draft_path(c, table, lengths, ints, lengths),
             lambda c: pk.tree_attention(x, c, table, lengths))
    for name, shape in (("value_codes", (2, 2, 16, 64)), ("key_scales", (4, 2, 8)), ("value_scales", (1,)),
                        ("key_codes", (8, 2, 16, 64))):
        for call in calls:
            c = _cache(pages=4)
            getattr(c, name).resize_(shape)
            with pytest.raises(ValueError, match="QuantizedKVCache"):
                call(c)


def test_workspace_sizes_belong_to_a_device(monkeypatch: pytest.MonkeyPatch) -> None:
    # Two fake devices whose plans differ, as GPUs with other SM counts' do.
    from piper_kernels.decoding import attention

    class Fake:
        current = 0

        def __init__(self, index):
            self.index = index

        def __enter__(self):
            self.before, Fake.current = Fake.current, self.index

        def __exit__(self, *_):
            Fake.current = self.before

    monkeypatch.setattr(torch.cuda, "device", Fake)
    monkeypatch.setattr(attention, "workspace_bytes", lambda *sizes: 1000 * Fake.current + len(sizes))
    attention._workspace_bytes.cache_clear()
    for _ in range(2):
        assert [attention._workspace_bytes(i, 1, 2, 1, 1, 64, 4096) for i in (0, 1)] == [6, 1006]
    attention._workspace_bytes.cache_clear()


def test_the_library_is_built_without_torch_and_the_binding_again_with_another(
    monkeypatch: pytest.MonkeyPatch, tmp_path
) -> None:
    # Fake compilers that write their output, and a fake torch.
    import importlib.util
    import subprocess
    from pathlib import Path

    path = Path(pk.__file__).resolve().parents[1] / "build.py"
    spec = importlib.util.spec_from_file_location("piper_build", path)
    build = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(build)
    for name in ("OUTPUT", "BINDING", "BINDING_TORCH"):
        monkeypatch.setattr(build, name, tmp_path / getattr(build, name).name)
    made = []

    class Compiler:
        def __init__(self, args, check=False):
            self.args, self.returncode = args, 0
            made.append(Path(args[args.index("-o") + 1]).name)
            Path(args[args.index("-o") + 1]).write_text("")

        def wait(self):
            return 0

    monkeypatch.setattr(subprocess, "Popen", Compiler)
    monkeypatch.setattr(subprocess, "run", Compiler)

    def outputs(**kw):
        made.clear()
        build.build(**kw)
        return {name for name in made if not name.endswith(".o")}

    version = [None]
    monkeypatch.setattr(build, "torch_version", lambda: version[0])
    assert outputs() == {"libpiper_b200.so"} and outputs() == set()
    version[0] = "2.0 True"
    assert outputs(library_only=True) == set()
    assert outputs() == {"decoding_binding.so"} and outputs() == set()
    version[0] = "2.1 True"
    assert outputs() == {"decoding_binding.so"} and outputs() == set()
    assert outputs(force=True) == {"libpiper_b200.so", "decoding_binding.so"}


def test_a_cache_that_wants_a_gradient_is_refused_where_it_would_lose_one() -> None:
    table, lengths = _batch()
    x, ints = torch.zeros(2, 2, 3, 64).half(), torch.zeros((2, 3), dtype=torch.int32)
    calls = {
        "write": lambda c: pk.write_kv_cache(c, x, x, table, lengths),
        "read": lambda c: pk.read_kv_cache(c, table, lengths, 2),
        "keep": lambda c: pk.keep_draft_path(c, table, lengths, ints, lengths),
        "attend": lambda c: pk.tree_attention(x, c, table, lengths),
    }
    learned = _cache(key_mean=torch.zeros(2, 64, requires_grad=True))
    scaled = _cache()
    scaled.value_scales.requires_grad_()
    for name, call in calls.items():
        with pytest.raises(RuntimeError, match="autograd"):
            call(scaled)
        # A softmax does not see the mean, and moved rows keep their codes.
        with pytest.raises(RuntimeError, match="autograd" if name in ("write", "read") else "no CPU"):
            call(learned)
        for cache in (scaled, learned):
            with torch.no_grad(), pytest.raises(RuntimeError, match="no CPU"):
                call(cache)


def test_registered_operators_check_their_arguments() -> None:
    # (On the CPU: the last check, after all others, is the device's.)
    ops = torch.ops.piper_kernels
    buffers, (table, lengths) = _cache().buffers, _batch()
    x, ints = torch.zeros(2, 2, 3, 64).half(), torch.zeros((2, 3), dtype=torch.int32)
    wide = table.long()

    def write(b=buffers, k=x, v=x, t=table, n=lengths):
        return ops.write_kv_cache(*b, k, v, t, n, None)

    def read(t=table, n=lengths, tokens=2, dtype=torch.float16):
        return ops.read_kv_cache(*buffers, t, n, None, tokens, dtype)

    def keep(t=table, n=lengths, path=ints, counts=lengths):
        return ops.keep_draft_path(*buffers[:4], t, n, path, counts)

    def attend(q=x, t=table, n=lengths, mask=None, scale=0.1):
        return ops.tree_attention(q, *buffers[:4], t, n, mask, scale)

    def verify(target=torch.zeros(2, 3, 5), draft=torch.zeros(2, 3, 5), noise=torch.zeros(2, 5)):
        return ops.verify_draft_tree(target, draft, ints.long(), ints, torch.zeros(2, 3), noise)

    for call, changes in (
        (write, [dict(t=wide), dict(n=lengths[:1]), dict(k=x[:, :1]), dict(v=x.float()), dict(b=_cache(d=128).buffers)]),
        (read, [dict(t=wide), dict(t=table[:1]), dict(tokens=0), dict(dtype=torch.float32)]),
        (keep, [dict(t=wide), dict(path=ints.long()), dict(counts=lengths[:1]), dict(n=lengths.long())]),
        (attend, [dict(t=wide), dict(n=lengths[:1]), dict(q=x[..., :32]), dict(mask=ints.long()[:, :2]), dict(scale=0.0)]),
        (verify, [dict(draft=torch.zeros(2, 3, 4)), dict(noise=torch.zeros(2, 4)), dict(target=torch.zeros(2, 3, 5).half())]),
    ):
        with pytest.raises(RuntimeError, match="no CPU or generic-GPU fallback"):
            call()
        for change in changes:
            with pytest.raises(ValueError):
                call(**change)
