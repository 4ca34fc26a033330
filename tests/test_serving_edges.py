"""The serving operators' host side at the edges of what it takes, without a GPU."""
import pytest
import torch

import lucid_b200 as lb
from lucid_b200 import _lib, paged
from test_paged import _cache, _held, _write, on_cpu  # noqa: F401


def test_a_batch_keeps_its_device_tensors(on_cpu):
    """A captured step reads the tensors' addresses: the bookkeeping writes into them."""
    cache = _cache(pages=40)
    batch = cache.batch(cache.new(2))
    _write(batch, [3, 5], [[1, 2, 3], [4, 5, 6, 7, 8]])
    kept = [batch.block_table, batch.lengths, batch.counts]
    other = cache.batch(cache.new())
    for step in range(12):
        if step == 4:
            cache.free(cache.fork(batch.sequences[0]))
        if step == 8:
            _write(other, [1], [[0]])
            other = cache.batch(cache.new())
        _write(batch, [1, step % 2], [[step], [step][:step % 2]])
        assert all(a is b for a, b in zip(kept, (batch.block_table, batch.lengths, batch.counts)))
        assert batch.lengths.tolist() == batch.host_lengths and batch.counts.tolist() == [1, step % 2]
        for row, s in zip(batch.block_table.tolist(), batch.sequences):
            assert row[:len(cache.pages(s))] == cache.pages(s)
    assert _held(cache, batch.sequences[0], 0) == [1, 2, 3, *range(12)]


def test_a_captured_batch_refuses_to_outgrow_its_table(on_cpu, monkeypatch):
    """With nothing changed; a new batch of the sequences goes on."""
    cache = _cache(pages=60)
    batch = cache.batch(cache.new(2))
    k = torch.zeros(2, 1, 1, 4, dtype=torch.bfloat16)
    batch.reserve(1)
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: True)
    batch.append(0, k, k)
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: False)
    batch.advance()
    room = batch.block_table.shape[1]
    child = cache.fork(batch.sequences[0])
    batch.reserve(room * 4 - 1)
    kept, free, refs = batch.block_table, cache.free_pages, list(cache._refs)
    with pytest.raises(_lib.LucidError, match="capture again"):
        batch.reserve([1, room * 4])
    assert batch.block_table is kept and cache.free_pages == free and cache._refs == refs
    assert cache.pages(child) and batch.host_lengths == [1, 1]
    batch = cache.batch(batch.sequences)
    batch.reserve([1, room * 4])
    batch.advance()
    assert batch.host_lengths == [2, room * 4 + 1]


def test_bookkeeping_in_and_out_of_inference_mode(on_cpu):
    """Tensors made in inference mode could not be written outside it."""
    cache = _cache(pages=40)
    a = cache.new(2)
    batch = cache.batch(a)
    with torch.inference_mode():
        _write(batch, [3, 5], [[1, 2, 3], [4, 5, 6, 7, 8]])
    _write(batch, [6, 1], [[4, 5, 6, 7, 8, 9], [9]])
    with torch.inference_mode():
        _write(batch, [1, 1], [[10], [10]])
    assert _held(cache, a[0], 1) == [2, 3, 4, 5, 6, 7, 8, 9, 10, 11] and batch.lengths.tolist() == [10, 7]


def test_without_query_heads_there_is_no_step(monkeypatch):
    """The new token's key would be neither solved nor cached."""
    monkeypatch.setattr(_lib, "_lib", object())
    monkeypatch.setattr(paged, "_pools", lambda k, x: (k.device, 0, 0, k.stride(), 0, x.stride()))
    t = torch.zeros(2, 0, 1, 64, dtype=torch.bfloat16)
    kv = torch.zeros(2, 2, 1, 64, dtype=torch.bfloat16)
    pool = torch.zeros(4, 2, 16, 64, dtype=torch.bfloat16)
    n = torch.zeros(2, dtype=torch.int32)
    with pytest.raises(ValueError, match="query"):
        lb.paged_decode_step(t, kv, kv, pool, pool, n[:, None], n, 0.1)


def test_the_entry_script_defines_what_it_runs():
    """python __graft_entry__.py smoke: everything that smoke() calls is there when the
    block at the script's end calls it."""
    import ast
    import os

    from conftest import ROOT
    with open(os.path.join(ROOT, "__graft_entry__.py")) as f:
        body = ast.parse(f.read()).body
    main = [i for i, n in enumerate(body) if isinstance(n, ast.If) and "__main__" in ast.unparse(n.test)]
    defined = [n.name for n in body[:main[0]] if isinstance(n, ast.FunctionDef)]
    everywhere = {n.name: n for n in body if isinstance(n, ast.FunctionDef)}
    assert "smoke" in defined and len(main) == 1
    reached, todo = set(), ["smoke", "build"]
    while todo:
        name = todo.pop()
        if name not in reached:
            reached.add(name)
            todo += [n.id for n in ast.walk(everywhere[name]) if isinstance(n, ast.Name) and n.id in everywhere]
    assert reached <= set(defined)


def _runs(code):
    import subprocess
    import sys

    from conftest import ROOT
    got = subprocess.run([sys.executable, "-c", code + "\nprint('fine')"], cwd=ROOT, capture_output=True, text=True, timeout=300)
    assert got.returncode == 0 and got.stdout.strip().endswith("fine"), got.stderr[-2000:]


def test_the_package_imports_on_a_torch_without_cuda():
    """Its C module lacks these names."""
    _runs("""
import torch
for name in ("_cuda_getCurrentRawStream", "_cuda_getDevice"):
    if hasattr(torch._C, name):
        delattr(torch._C, name)
import lucid_b200 as lb
t = torch.zeros(4, 1, 4, 4, dtype=torch.bfloat16)
for call in (lambda: lb.copy_pages(t, t, [0], [1]), lambda: lb.token_logprobs(torch.zeros(2, 5), None)):
    try:
        call()
    except RuntimeError as e:
        assert "no CPU fallback" in str(e), e
    else:
        raise AssertionError
""")


def test_the_cache_keeps_its_books_without_a_gpu():
    """Asking for the capture of a stream raises where CUDA cannot be used."""
    _runs("""
import torch
def none():
    raise RuntimeError("no CUDA here")
torch.cuda.is_current_stream_capturing = none
import lucid_b200 as lb
cache = lb.PagedCache(1, 1, 4, 12, 4, device="cpu")
batch = cache.batch(cache.new(2))
batch.reserve([3, 5])
batch.advance()
cache.free(batch.sequences[0])
assert cache.free_pages == 10 and cache.length(batch.sequences[1]) == 5
""")


def test_token_logprobs_refuse_forward_mode():
    """The tangent of the logits would be dropped."""
    from torch.autograd import forward_ad
    x = torch.randn(2, 5, requires_grad=False)
    with forward_ad.dual_level():
        for logits in (forward_ad.make_dual(x, torch.ones_like(x)), forward_ad.make_dual(x.clone().requires_grad_(), x)[:, :4]):
            with pytest.raises(NotImplementedError, match="forward mode"):
                lb.token_logprobs(logits, None)
            with torch.no_grad(), pytest.raises(NotImplementedError, match="forward mode"):
                lb.token_logprobs(logits, None)
        with pytest.raises(RuntimeError, match="no CPU fallback"):
            lb.token_logprobs(x, None)
    with pytest.raises(NotImplementedError, match="forward mode"):
        torch.func.jvp(lambda z: lb.token_logprobs(z, None).entropy, (x,), (x,))


def test_a_negative_count_of_new_sequences(on_cpu):
    """It would hand out the numbers of living sequences again."""
    cache = _cache()
    a, b = cache.new(2)
    _write(cache.batch([b]), [2], [[1, 2]])
    for bad in (-1, -2):
        with pytest.raises(ValueError, match="count"):
            cache.new(bad)
    assert cache.new(0) == [] and cache.new() == [b + 1] and _held(cache, b, 0) == [1, 2]


def test_check_status_refuses_a_capture(monkeypatch):
    """It waits for the devices whose words it reads, which would spoil the capture."""
    import ctypes
    word = ctypes.c_int32(0)
    watch = _lib._StatusWatch()
    waited = []
    monkeypatch.setattr(torch.cuda, "synchronize", waited.append)
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: True)
    watch.wait_all()                                  # no words: nothing to wait for
    watch.words[0] = (None, word, 0)
    with pytest.raises(_lib.LucidError, match="outside the capture"):
        watch.wait_all()
    assert not waited
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: False)
    word.value = 4 | 16 << 20
    with pytest.raises(_lib.LucidError, match="paged decoding"):
        watch.wait_all()
    watch.wait_all()
    assert waited == [0, 0]


def test_another_batch_grows_a_captured_batchs_sequence(on_cpu, monkeypatch):
    """Its reserved pages alone are more than the captured table holds."""
    cache = _cache(pages=60)
    batch = cache.batch(cache.new())
    k = torch.zeros(1, 1, 1, 4, dtype=torch.bfloat16)
    batch.reserve(1)
    with monkeypatch.context() as m:
        m.setattr(torch.cuda, "is_current_stream_capturing", lambda: True)
        batch.append(0, k, k)
    batch.advance()
    kept, other = batch.block_table, cache.batch(batch.sequences)
    other.reserve(4 * kept.shape[1] + 4)
    with pytest.raises(_lib.LucidError, match="capture again"):
        batch.reserve(1)
    assert batch.block_table is kept
