"""The paged key/value cache without a GPU: the index arithmetic of its kernels compiled for the host, and the library's host side on
a CUDA runtime of host memory (fake_cudart.cpp): what it refuses, and what its launches get."""
import ctypes as C
import os
import subprocess
import sys

import numpy as np
import pytest

from test_host_paths import LAUNCH, _fake, fake_runtime  # noqa: F401 (a fixture)

HERE = os.path.dirname(os.path.abspath(__file__))
SCENARIOS = {}

INDEX = r"""
#include "kv_index.h"
using namespace mb;
extern "C" {
int seq(const int *off, const int *len, int s, int rows, long long cap, int *out) {
    KvSeq q; const bool ok = kv_seq(off, len, s, rows, cap, &q); out[0] = q.begin; out[1] = q.n; out[2] = q.len; return ok;
}
int sees(int pos, int j, int window, int sinks) { return kv_sees(pos, j, window, sinks); }
int tiles(int p0, int p1, int window, int sinks, int tile, int *out, int cap) {
    const KvTiles t = kv_tiles(p0, p1, window, sinks, tile);
    for (int i = 0; i < t.count && i < cap; i++) out[i] = t.at(i);
    return t.count;
}
int groups(int p0, int p1, int window, int sinks, int *out, int cap) {
    const KvGroups t = kv_groups(p0, p1, window, sinks);
    for (int i = 0; i < t.count && i < cap; i++) out[i] = t.at(i);
    return t.count;
}
}
"""


@pytest.fixture(scope="module")
def index(tmp_path_factory):
    out = tmp_path_factory.mktemp("kv_index")
    (out / "index.cpp").write_text(INDEX)
    subprocess.run(["g++", "-std=c++17", "-O1", "-fPIC", "-shared", "-fsanitize=undefined", "-fno-sanitize-recover", "-I",
                    os.path.join(HERE, "..", "mynah-asr_b200", "csrc"), str(out / "index.cpp"), "-o", str(out / "index.so")], check=True)
    return C.CDLL(str(out / "index.so"))


def test_sequences_of_tables(index):
    """Whatever the tables say, what comes out lies inside of the call's buffers."""
    top = 2 ** 31 - 1
    numbers = [0, 1, -1, 5, 9, 10, 11, top, -top - 1, top - 1]
    out, cap = (C.c_int * 3)(), 96
    for b in numbers:
        for e in numbers:
            for n in numbers:
                off, length = (C.c_int * 2)(b, e), (C.c_int * 1)(n)
                ok = index.seq(off, length, 0, 10, C.c_longlong(cap), out)
                assert bool(ok) == (0 <= b <= e <= 10 and 0 <= n <= cap)
                if ok:
                    assert list(out) == [b, e - b, n]
                else:
                    assert out[1] == out[2] == 0
                ok = index.seq(None, length, 0, 10, C.c_longlong(cap), out)
                assert bool(ok) == (0 <= n <= cap) and (not ok or list(out) == [0, 1, n])


@pytest.mark.parametrize("tile", [32, 128])
def test_tiles_cover_what_is_seen(index, tile):
    """The tiles of rows at [p0, p1]: in order, none twice, every visible key in one of them, and none of a window's without one."""
    out = (C.c_int * 4096)()
    for window in (0, 1, 5, tile - 1, tile, tile + 1, 3 * tile + 7, 2 ** 31 - 1):
        for sinks in ((0, 1, tile, tile + 1, 5 * tile, 2 ** 31 - 1) if window else (0,)):
            for p0 in (-7, -1, 0, 1, tile - 1, tile, 4 * tile, 9 * tile + 3, 20 * tile):
                for more in (0, 1, tile - 1, tile, 2 * tile + 5):
                    p1 = p0 + more
                    n = index.tiles(p0, p1, window, sinks, tile, out, 4096)
                    got = list(out[:n])
                    rows = [p for p in {p0, p0 + more // 2, p1} if p >= 0]
                    need = {j // tile for p in rows for j in range(p + 1) if index.sees(p, j, window, sinks)}
                    assert got == sorted(set(got)) and need <= set(got), (window, sinks, p0, p1, got)
                    assert all(0 <= t <= max(p1, 0) // tile for t in got)
                    if window and more == 0 and p0 >= 0:
                        assert set(got) - need <= {t for t in got if t < min(sinks, p0 + 1) / tile} | need
    top = 2 ** 31 - 1
    assert index.tiles(top - 5, top - 1, 64, 4, tile, out, 4096) in (2, 3, 4)
    assert index.tiles(top - 5, top - 1, 64, top, tile, out, 4096) == (top - 1) // tile + 1


def test_groups_cover_what_is_seen(index):
    """The groups of 32 keys of rows at [p0, p1]: in order, none twice, every visible key in one, and none that no row sees."""
    out = (C.c_int * 4096)()
    for window in (0, 1, 5, 31, 32, 33, 128, 391, 2 ** 26):
        for sinks in ((0, 1, 32, 33, 160, 2 ** 26) if window else (0,)):
            for p0 in (-7, -1, 0, 1, 31, 32, 33, 127, 128, 515, 2560):
                for more in (0, 1, 31, 32, 127, 261):
                    p1 = p0 + more
                    n = index.groups(p0, p1, window, sinks, out, 4096)
                    got = list(out[:n])
                    need = {j // 32 * 32 for p in range(max(p0, 0), p1 + 1) for j in ([*range(min(sinks, p + 1)), *range(max(p - window + 1, 0), p + 1)] if window else range(p + 1))}
                    assert got == sorted(set(got)) and need <= set(got), (window, sinks, p0, p1, got)
                    assert all(j % 32 == 0 and 0 <= j <= max(p1, 0) for j in got)
                    if p0 >= 0:                               # (the group between the first tokens and the window may come too, where they meet)
                        assert len(set(got) - need) <= 1
    top = 2 ** 26 - 1
    assert index.groups(top - 5, top, 64, 4, out, 4096) in (3, 4) and index.groups(0, top, 2 ** 26, 2 ** 26, out, 4096) == 2 ** 21


def test_numbers_beyond_32_bits(pkg):
    """What ctypes would cut to 32 bits is refused: 2^32 + 8 pages are not eight."""
    good = dict(n_heads=4, n_kv_heads=2, head_dim=64, page_size=16, n_pages=8, window=64, n_sinks=1)
    for name in good:
        for more in (2 ** 32, -2 ** 32, 2 ** 40):
            with pytest.raises(ValueError, match=name):
                pkg.KvCache(**dict(good, **{name: good[name] + more}))


def test_integration_example(tmp_path):
    """The layer shown to hosts is C that compiles against the header, and waits wherever rows pass from one stream to another."""
    with open(os.path.join(HERE, "..", "INTEGRATION.md")) as f:
        code = f.read().split("## 4b.")[1].split("```c\n")[1].split("```")[0]
    (tmp_path / "layer.c").write_text('#include <stdio.h>\n#include "mynah_b200.h"\nvoid layer(const mynah_b200_qmat *w_qkv, const mynah_b200_qmat *w_out, '
                                      "const float *h, float *x, float *q, float *y, long long ld, int n_seq, int n_rows, const int *row_off, const int *kv_len, "
                                      "const int *page_table, int max_pages, void *stream) {\n" + code + "}\n")
    subprocess.run(["gcc", "-std=c11", "-Wall", "-Werror", "-fsyntax-only", "-I", os.path.join(HERE, "..", "include"), str(tmp_path / "layer.c")], check=True)
    calls = [line.split("mynah_b200_")[1].split("(")[0] for line in code.splitlines() if "bad |" in line or "int bad" in line]
    assert calls == ["qmat_mul_device", "qmat_sync", "kv_append", "kv_attend", "kv_sync", "qmat_mul_device", "qmat_sync"]


def test_registers_are_looked_at_by_the_build():
    """A compiler that gives the prompts' kernel another number of registers than it deals out is found by the build."""
    from importlib.util import module_from_spec, spec_from_file_location
    spec = spec_from_file_location("mynah_build", os.path.join(HERE, "..", "mynah-asr_b200", "build.py"))
    build = module_from_spec(spec)
    spec.loader.exec_module(build)
    report = "".join("ptxas info    : Compiling entry function '_ZN2mb15kv_chunk_kernelILi%dELi%dELb0EEEv' for 'sm_100a'\nptxas info    : Function properties for x\n"
                     "    0 bytes stack frame\nptxas info    : Used %d registers, used 1 barriers\n" % (d, f, {64: 128, 128: 168}[d]) for d in (64, 128) for f in range(3))
    assert build.missing_registers("kv_chunk.cu", report) == [] and build.missing_registers("kv.cu", "") == []
    assert len(build.missing_registers("kv_chunk.cu", report.replace("168", "160", 1))) == 1
    assert len(build.missing_registers("kv_chunk.cu", report.replace("128 registers", "126 registers"))) == 3
    assert len(build.missing_registers("kv_chunk.cu", "")) == 2
    with open(os.path.join(build.CSRC, "kv_chunk.cu")) as f:
        assert "REGS = SOFT == 8 ? 168 : 128" in f.read()


# ------------------------------------------------------------------------------------------- in the child process
def scenario(f):
    SCENARIOS[f.__name__] = f
    return f


@pytest.mark.parametrize("name", ["kv_refuses", "kv_gives_back", "kv_launches", "kv_failed_calls"])
def test_kv_host(fake_runtime, name):  # noqa: F811
    env = dict(os.environ, LD_LIBRARY_PATH=fake_runtime + ":" + os.environ.get("LD_LIBRARY_PATH", ""), OMP_NUM_THREADS="1")
    r = subprocess.run([sys.executable, os.path.abspath(__file__), name], env=env, capture_output=True, text=True, timeout=300)
    assert r.returncode == 0, r.stdout + r.stderr


@pytest.mark.parametrize("name", ["kv_limits", "kv_overlaps", "kv_beside_a_torch_without_cuda"])
def test_kv_host_limits(fake_runtime, name):  # noqa: F811
    test_kv_host(fake_runtime, name)


def _config(pkg, **more):
    c = pkg.KvConfig()
    pkg.lib().mynah_b200_kv_config_default(C.byref(c))
    for name, value in dict(dict(n_heads=4, n_kv_heads=2, head_dim=64, n_pages=8), **more).items():
        setattr(c, name, value)
    return c


def _dev(n):
    """n bytes of the fake device's memory."""
    L, p = C.CDLL("libcudart.so.12"), C.c_void_p()
    assert L.cudaMalloc(C.byref(p), C.c_size_t(n)) == 0
    return p.value


def _batch(pkg, n_seq=2, n_rows=2, row_off=None, kv_len=0, page_table=0, max_pages=4):
    return pkg.KvBatchStruct(n_seq, n_rows, row_off, kv_len, page_table, max_pages)


@scenario
def kv_refuses(pkg, fake):
    """Every refusal comes with its reason, before anything is launched or allocated."""
    L = pkg.lib()
    nan, inf = float("nan"), float("inf")
    before = fake.fake_device_bytes()
    for more in (dict(fmt=pkg.MYNAH_Q8), dict(fmt=77), dict(n_heads=0), dict(n_kv_heads=0), dict(n_heads=5), dict(n_heads=-4), dict(n_heads=130),
                 dict(head_dim=8), dict(head_dim=72), dict(head_dim=144), dict(head_dim=0), dict(page_size=12), dict(page_size=4), dict(page_size=512),
                 dict(page_size=0), dict(n_pages=0), dict(n_pages=2 ** 27), dict(rotary_dim=4), dict(rotary_dim=72), dict(rotary_dim=-8),
                 dict(rotary_dim=8, rope_theta=0.0), dict(rotary_dim=8, rope_theta=nan), dict(window=-1), dict(n_sinks=2), dict(window=3, n_sinks=-1),
                 dict(scale=-1.0), dict(scale=nan), dict(scale=inf), dict(norm_eps=nan, q_norm=(C.c_float * 64)()), dict(norm_eps=-1.0, k_norm=(C.c_float * 64)()),
                 dict(q_norm=(C.c_float * 64)(*([1.0] * 63 + [nan]))), dict(rotary_dim=8, inv_freq=(C.c_double * 4)(1, 2, inf, 3))):
        assert L.mynah_b200_kv_create(C.byref(_config(pkg, **more))) is None, more
        assert b"kv_create" in L.mynah_b200_last_error(), more
    assert L.mynah_b200_kv_create(None) is None and fake.fake_device_bytes() == before
    h = L.mynah_b200_kv_create(C.byref(_config(pkg, rotary_dim=64)))
    assert h
    seen = []
    cb = LAUNCH(lambda name, args, recorded: seen.append(name))
    fake.fake_on_launch(cb)
    lens, table, off, rows = _dev(64), _dev(256), _dev(64), _dev(1 << 16)
    good = dict(kv_len=lens, page_table=table)
    call = lambda b, q=rows, ldq=256, out=rows, ldo=256: L.mynah_b200_kv_attend(h, C.addressof(b), q, ldq, out, ldo, None)  # noqa: E731
    host = np.zeros(4096, np.float32)
    for b in (dict(good, n_seq=-1), dict(good, n_rows=-1), dict(good, n_rows=2 ** 30 + 1), dict(good, n_seq=2 ** 31 - 1, n_rows=2 ** 31 - 1, row_off=off),
              dict(good, max_pages=2 ** 22 + 1), dict(good, kv_len=None), dict(good, page_table=None), dict(good, max_pages=0),
              dict(good, max_pages=2 ** 28), dict(good, n_seq=3), dict(good, kv_len=lens + 2), dict(good, row_off=off + 1),
              dict(good, kv_len=host.ctypes.data), dict(good, page_table=host.ctypes.data), dict(good, row_off=host.ctypes.data)):
        assert call(_batch(pkg, **b)) == -1, b
        assert b"kv_attend" in L.mynah_b200_last_error()
    b = _batch(pkg, **good)
    for more in (dict(q=None), dict(q=rows + 4), dict(q=host.ctypes.data), dict(ldq=255), dict(ldq=-256), dict(ldq=257), dict(ldq=2 ** 50), dict(out=None),
                 dict(out=rows + 8), dict(out=host.ctypes.data), dict(ldo=128), dict(ldo=258)):
        assert call(b, **more) == -1, more
    at = C.addressof(b)
    for bad in range(4):
        for value, ld in ((None, 256), (rows + 4, 256), (rows, 100), (host.ctypes.data, 256)):
            args = [x for i in range(4) for x in ((value, ld) if i == bad else (rows, 256))]
            assert L.mynah_b200_kv_append(h, at, *args, None) == -1
            assert b"kv_append" in L.mynah_b200_last_error()
    assert L.mynah_b200_kv_append(None, at, *([rows, 256] * 4), None) == L.mynah_b200_kv_attend(h, None, rows, 256, rows, 256, None) == -1
    assert L.mynah_b200_kv_sync(None, None) == -1 and L.mynah_b200_kv_pages(h, None, None) == -1
    for empty in (dict(good, n_seq=0), dict(good, n_rows=0, n_seq=0), dict(good, n_rows=0, row_off=off)):
        assert call(_batch(pkg, **empty)) == 0
    assert not seen
    assert call(b) == 0 and len(seen) == 1
    assert L.mynah_b200_kv_append(h, at, *([rows, 256] * 4), None) == 0 and len(seen) == 2
    assert L.mynah_b200_kv_sync(h, None) == 0
    L.mynah_b200_kv_free(h)
    L.mynah_b200_kv_free(None)


@scenario
def kv_gives_back(pkg, fake):
    """Whatever fails while a handle is made, nothing stays allocated; a handle that is freed gives all of it back."""
    L = pkg.lib()
    before = fake.fake_device_bytes()
    for name, most in ((b"cudaMalloc", 3), (b"cudaStreamCreate", 1), (b"cudaMemsetAsync", 3)):
        for nth in range(1, most + 1):
            fake.fake_fail(name, nth)
            assert L.mynah_b200_kv_create(C.byref(_config(pkg))) is None
            assert fake.fake_failed() and b"kv_create" in L.mynah_b200_last_error()
            assert fake.fake_device_bytes() == before, name
    h = L.mynah_b200_kv_create(C.byref(_config(pkg)))
    assert fake.fake_device_bytes() - before >= 2 * 8 * 16 * 2 * 64 * 2
    L.mynah_b200_kv_free(h)
    assert fake.fake_device_bytes() == before


@scenario
def kv_launches(pkg, fake):
    """A recorded call and a plain one are one launch each, allocate nothing and leave another thread's recording alone."""
    L = pkg.lib()
    w = (C.c_float * 64)(*range(64))
    fake.fake_foreign_capture(1)
    h = L.mynah_b200_kv_create(C.byref(_config(pkg, q_norm=w, rotary_dim=16)))
    assert h and fake.fake_broken_captures() == 0
    fake.fake_foreign_capture(0)
    lens, table, off, rows = _dev(64), _dev(256), _dev(64), _dev(1 << 16)
    seen = []
    cb = LAUNCH(lambda name, args, recorded: seen.append(name))
    fake.fake_on_launch(cb)
    held, mallocs, count = fake.fake_device_bytes(), fake.fake_calls(b"cudaMalloc"), pkg.launch_count()
    for row_off in (None, off):
        b = _batch(pkg, kv_len=lens, page_table=table, row_off=row_off)
        assert L.mynah_b200_kv_append(h, C.addressof(b), *([rows, 256] * 4), None) == 0
        assert L.mynah_b200_kv_attend(h, C.addressof(b), rows, 256, rows, 256, None) == 0
    assert len(seen) == 4 and pkg.launch_count() == count + 4
    assert fake.fake_device_bytes() == held and fake.fake_calls(b"cudaMalloc") == mallocs
    assert fake.fake_pending() == 1                      # asynchronous
    assert L.mynah_b200_kv_sync(h, None) == 0 and fake.fake_pending() == 0
    L.mynah_b200_kv_free(h)


@scenario
def kv_failed_calls(pkg, fake):
    """A launch or a copy that fails is that call's error and not the next one's."""
    L = pkg.lib()
    h = L.mynah_b200_kv_create(C.byref(_config(pkg)))
    lens, table, rows = _dev(64), _dev(256), _dev(1 << 16)
    b = _batch(pkg, kv_len=lens, page_table=table)
    for call in (lambda: L.mynah_b200_kv_append(h, C.addressof(b), *([rows, 256] * 4), None),
                 lambda: L.mynah_b200_kv_attend(h, C.addressof(b), rows, 256, rows, 256, None)):
        fake.fake_fail(b"cudaLaunchKernel", 1)
        assert call() == -1 and fake.fake_failed()
        assert call() == 0
    fake.fake_fail(b"cudaMemcpyAsync", 1)
    assert L.mynah_b200_kv_sync(h, None) == -1 and L.mynah_b200_kv_sync(h, None) == 0
    L.mynah_b200_kv_free(h)


@scenario
def kv_limits(pkg, fake):
    """As many sequences as a warp can look through within the limit on waits, and not one more."""
    L = pkg.lib()
    h = L.mynah_b200_kv_create(C.byref(_config(pkg)))
    lens, table, off, rows = _dev(4 << 16), _dev(4 << 18), _dev((4 << 16) + 4), _dev(256)
    seen = []
    cb = LAUNCH(lambda name, args, recorded: seen.append(name))
    fake.fake_on_launch(cb)
    for n, row_off, n_rows, ok in ((1 << 16, off, 1, True), (1 << 16, None, 1 << 16, True), ((1 << 16) + 1, off, 1, False), ((1 << 16) + 1, None, 1 << 17, False)):
        b, before = _batch(pkg, n_seq=n, n_rows=n_rows, row_off=row_off, kv_len=lens, page_table=table, max_pages=4), len(seen)
        for call in (lambda: L.mynah_b200_kv_append(h, C.addressof(b), *([rows, 256] * 4), None), lambda: L.mynah_b200_kv_attend(h, C.addressof(b), rows, 256, rows, 256, None)):
            assert call() == (0 if ok else -1)
            assert ok or b"sequences" in L.mynah_b200_last_error()
        assert len(seen) == before + 2 * ok
    L.mynah_b200_kv_free(h)


@scenario
def kv_overlaps(pkg, fake):
    """Results that would be read as other rows' input are refused; the same rows, and columns side by side, are not."""
    L = pkg.lib()
    h = L.mynah_b200_kv_create(C.byref(_config(pkg)))                # rows of 256 and 128 f32 values
    lens, table, at = _dev(64), _dev(256), _dev(1 << 16) + (1 << 14)
    b = _batch(pkg, n_seq=3, n_rows=3, kv_len=lens, page_table=table)
    far = _dev(1 << 14)
    for ld, out, ldo, ok in ((256, at, 256, True), (512, at, 512, True), (512, at + 256 * 4, 512, True), (512, at - 256 * 4, 512, True), (256, at + 3 * 1024, 256, True),
                             (256, at - 3 * 1024, 256, True), (256, far, 512, True), (512, at + 2 * 2048 + 1024, 256, True),
                             (256, at + 16, 256, False), (256, at + 1024, 256, False), (256, at - 2048, 256, False), (512, at + 255 * 4 - 12, 512, False),
                             (512, at + 257 * 4 - 4 + 16, 512, False), (256, at, 512, False), (512, at + 2048, 256, False), (512, at + 2 * 2048 + 1008, 256, False)):
        assert (L.mynah_b200_kv_attend(h, C.addressof(b), at, ld, out, ldo, None) == 0) == ok, (ld, out - at, ldo)
        assert ok or b"overlaps" in L.mynah_b200_last_error()
        assert (L.mynah_b200_kv_append(h, C.addressof(b), at, ld, far, 128, far, 128, out if out != far else far + 8192, ldo, None) == 0) == ok
    one = _batch(pkg, n_seq=1, n_rows=1, kv_len=lens, page_table=table)
    for out, ldo, ok in ((at, 256, True), (at, 512, True), (at + 1024, 256, True), (at + 1008, 512, False), (at - 1008, 256, False)):
        assert (L.mynah_b200_kv_attend(h, C.addressof(one), at, 260, out, ldo, None) == 0) == ok, (out - at, ldo)
    for k, v, ok in ((at + 1024, at + 1536, True), (at + 1024, at + 1008, False), (at + 512, at + 1536, False), (at - 512, at + 1024, True), (at - 496, at + 1024, False)):
        assert (L.mynah_b200_kv_append(h, C.addressof(b), at, 512, k, 512, v, 512, at, 512, None) == 0) == ok, (k - at, v - at)
    L.mynah_b200_kv_free(h)


@scenario
def kv_beside_a_torch_without_cuda(pkg, fake):
    """A process may have a torch that knows no CUDA, or none: the tensors are another library's, the stream is the handle's own."""
    import types

    def no_cuda():
        raise AssertionError("Torch not compiled with CUDA enabled")

    stub = types.SimpleNamespace(cuda=types.SimpleNamespace(is_available=lambda: False, current_device=no_cuda, current_stream=no_cuda))
    for torch in (stub, None):
        if torch is None:
            sys.modules.pop("torch", None)
        else:
            sys.modules["torch"] = torch
        cache = pkg.KvCache(4, 2, 64, 16, 8, fmt=pkg.F32)
        cache.sync()
        cache.close()


if __name__ == "__main__":
    sys.path.insert(0, HERE)
    import conftest
    SCENARIOS[sys.argv[1]](conftest.load_package(), _fake())
