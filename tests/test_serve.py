"""CPU checks of the batched-serving entries: struct layout, refusals that need no device."""
import contextlib
import ctypes as C
import os
import shutil
import subprocess

import pytest
import torch

from loom_b200 import LoomCudaError, _lib, serve


def test_descriptors_match_the_header(tmp_path):
    """Size of each descriptor and the offset of each field."""
    if not shutil.which("gcc"):
        pytest.skip("no C compiler")
    names = {"loom_attn_shared_desc": _lib.AttnSharedDesc, "loom_lora_desc": _lib.LoraDesc,
             "loom_verify_desc": _lib.VerifyDesc}
    lines, want = [], []
    for n, cls in names.items():
        lines.append('printf("%%zu\\n", sizeof(%s));' % n)
        want.append(C.sizeof(cls))
        for f, _ in cls._fields_:
            lines.append('printf("%%zu\\n", offsetof(%s, %s));' % (n, f))
            want.append(getattr(cls, f).offset)
    src = tmp_path / "sz.c"
    src.write_text('#include <stdio.h>\n#include <stddef.h>\n#include "%s"\nint main(void){%s return 0;}\n' % (
        _lib.HEADER, " ".join(lines)))
    exe = tmp_path / "sz"
    subprocess.run(["gcc", "-o", str(exe), str(src)], check=True)
    assert [int(v) for v in subprocess.run([str(exe)], capture_output=True, text=True, check=True).stdout.split()] == want


def test_workspace_sizes_and_bad_descriptors():
    L = _lib.lib()
    good = dict(type=30, scale=0.1, n_seqs=4, n_rows=9, n_heads=32, n_kv_heads=4, head_dim=128, q_stride=4096,
                out_stride=4096, prefix_len=1000, prefix_pos_stride=512, prefix_head_stride=128, own_cap=300,
                own_pos_stride=512, own_head_stride=128, own_seq_stride=300 * 512)
    ws = lambda **kw: L.loom_cuda_attn_shared_workspace(C.byref(_lib.AttnSharedDesc(**{**good, **kw})))  # noqa: E731
    assert ws() > 0
    assert ws(type=0) > 0 and ws(type=8) == 0 and ws(n_kv_heads=5) == 0 and ws(head_dim=257) == 0
    assert ws(n_heads=0) == 0 and ws(prefix_len=1 << 40) == 0 and ws(n_rows=1 << 40) == 0
    lora = lambda **kw: L.loom_cuda_lora_workspace(C.byref(_lib.LoraDesc(**{**dict(  # noqa: E731
        type=1, n_rows=5, n_in=64, n_out=32, n_adapters=2, max_rank=8, x_stride=64, base_stride=32, out_stride=32,
        a_row_stride=64, a_adapter_stride=512, b_row_stride=8, b_adapter_stride=256), **kw})))
    assert lora() > 0 and lora(type=12) == 0 and lora(n_in=0) == 0 and lora(max_rank=5000) == 0
    ver = lambda **kw: L.loom_cuda_verify_workspace(C.byref(_lib.VerifyDesc(**{**dict(  # noqa: E731
        type=0, n_seqs=2, n_rows=5, vocab=100, logits_stride=100, probs_stride=0), **kw})))
    assert ver() > 0 and ver(type=2) == 0 and ver(vocab=0) == 0 and ver(vocab=1 << 30) == 0


def test_entries_decline_before_init():
    L = _lib.lib()
    d = _lib.VerifyDesc(0, 1, 1, 4, 4, 0)
    assert L.loom_cuda_verify(C.byref(d), *[None] * 10, 0, None) == _lib.DECLINED
    assert "init" in _lib.last_error()
    assert L.loom_cuda_lora(C.byref(_lib.LoraDesc()), *[None] * 9, 0, None) == _lib.DECLINED
    assert L.loom_cuda_attn_shared(C.byref(_lib.AttnSharedDesc()), *[None] * 9, 0, None) == _lib.DECLINED


def test_host_tensors_are_refused():
    z, i = torch.zeros, torch.zeros(2, dtype=torch.int32)
    with pytest.raises(LoomCudaError, match="cuda"):
        serve.attn_shared(z(1, 2, 8), z(4, 1, 8), z(4, 1, 8), z(1, 4, 1, 8), z(1, 4, 1, 8), i, i[:1], 1.0)
    with pytest.raises(LoomCudaError, match="cuda"):
        serve.lora(z(1, 4), z(1, 2, 4), z(1, 3, 2), i[:1], z(1), i[:1])
    with pytest.raises(LoomCudaError, match="cuda"):
        serve.verify(z(1, 4), i[:1], i, z(1))


class FakeTorch:
    """The parts of torch that a call's allocations need: which stream is current when memory is asked for, and which
    streams are captured."""
    uint8 = torch.uint8

    def __init__(self, captured=()):
        self.now, self.made, self.cuda, self.captured = 1, [], self, set(captured)

    def ExternalStream(self, st, device=None):
        return st

    def default_stream(self, dev):
        return 0

    def current_stream(self, dev=None):
        return self.now

    @contextlib.contextmanager
    def stream(self, st):
        was, self.now = self.now, st
        yield
        self.now = was

    def empty(self, shape, dtype=None, device=None):
        self.made.append((self.now, shape))
        return self

    def numel(self):
        return 1

    def record_stream(self, st):
        pass

    def data_ptr(self):
        return 64


@pytest.fixture
def fake(monkeypatch):
    def use(**kw):
        f = FakeTorch(**kw)
        monkeypatch.setattr(serve, "torch", f)
        monkeypatch.setattr(serve, "_stream", lambda dev: f.now)
        monkeypatch.setattr(serve, "_capturing", lambda: f.now in f.captured)
        monkeypatch.setattr(serve, "_kept", {})
        monkeypatch.setattr(serve, "_up", lambda op, dev: None)
        return f
    return use


def run_on(stream):
    serve._run("op", lambda *a: _lib.OK, lambda d: 1000, None, (), 0, stream)


def test_scratch_belongs_to_the_stream_of_the_call(fake):
    """Memory of the current stream's pool may still be in use by kernels that wait on it."""
    f = fake()
    run_on(7)
    run_on(0)
    assert f.made == [(7, 1000), (0, 1000)] and f.now == 1
    run_on(None)
    run_on(1)
    assert f.made[2:] == [(1, serve._KEEP)]


def test_scratch_of_captured_calls(fake):
    """A graph keeps what torch gives the capture; a stream captured behind torch's back has no such memory."""
    f = fake(captured=[1])
    run_on(None)
    assert f.made == [(1, 1000)]
    f = fake(captured=[1, 7])
    run_on(7)
    assert f.made == [(7, 1000)]
    f = fake(captured=[7])
    with pytest.raises(LoomCudaError, match="captured"):
        run_on(7)
    assert f.made == []


def test_shared_memory_limit_of_two_threads(tmp_path):
    """The larger limit stays, whichever thread comes back from the driver last."""
    if not shutil.which("g++"):
        pytest.skip("no C++ compiler")
    (tmp_path / "t.cc").write_text('''
#include "smem_limit.h"
#include <chrono>
#include <cstdio>
#include <thread>
int main() {
    loom::SmemLimit l;
    size_t set = 0;
    int asked = 0;
    auto nap = [](int ms) { std::this_thread::sleep_for(std::chrono::milliseconds(ms)); };
    std::thread large([&] { l.need(0, 200, [&](size_t n) { set = n; asked++; nap(400); return 0; }); });
    std::thread small([&] { nap(100); l.need(0, 100, [&](size_t n) { nap(100); set = n; asked++; return 0; }); });
    large.join();
    small.join();
    l.need(0, 200, [&](size_t n) { set = n; asked++; return 0; });
    const int refused = l.need(0, 300, [&](size_t) { return 7; });
    const int again = l.need(0, 300, [&](size_t n) { set = n; return 0; });
    std::printf("%zu %d %d %d\\n", set, asked, refused, again);
    return set == 300 && asked == 1 && refused == 7 && again == 0 ? 0 : 1;
}
''')
    src = os.path.join(os.path.dirname(_lib.HEADER), "..", "loom_b200", "csrc")
    subprocess.run(["g++", "-std=c++17", "-O1", "-pthread", "-I", src, "-o", str(tmp_path / "t"), str(tmp_path / "t.cc")], check=True)
    r = subprocess.run([str(tmp_path / "t")], capture_output=True, text=True, timeout=60)
    assert r.returncode == 0, r.stdout
