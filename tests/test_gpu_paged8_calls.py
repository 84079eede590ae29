"""GPU tests of the native module that makes the paged cache's short calls: it makes them (a wrapper goes on in Python, with the same
result, where it does not), and other threads run while a call waits for the GPU."""
import ctypes
import subprocess
import threading
import time

import pytest
import torch

from test_gpu_books import _books

pytestmark = pytest.mark.gpu
BF, F32, E4, I8, I32 = torch.bfloat16, torch.float32, torch.float8_e4m3fn, torch.int8, torch.int32


def _calls(dev, code):
    """{what: a call by the public functions} of each function of the module over a pool of `code`."""
    import tabicl_mi355_paged as paged
    table, n, free, fc, _ = _books(dev, 3, [50, 300, 0, 17], 40, 16, spare=90)
    P, H, D, R = free.numel(), 2, 64, 16
    eight = code in (E4, I8)
    kp, vp = (torch.zeros(P, H, R, D, device=dev).to(code) for _ in range(2))
    scales = torch.ones(P, H, 2, device=dev) if eight else None
    count = torch.tensor([20, 100, 33, 1], dtype=I32, device=dev)
    dtype = BF if eight else code
    x = torch.ones(160, H, D, dtype=dtype, device=dev)
    slots, starts = paged.paged_slots(table, n, count, 160, P, R)
    bnd, bs = torch.zeros(P, H, 2, D, dtype=I8, device=dev), torch.zeros(P, H, device=dev)
    q = torch.ones(4, 2 * H, 3, D, dtype=dtype, device=dev)
    out = torch.empty(4, 3, 2 * H, D, dtype=dtype, device=dev).transpose(1, 2)
    index = torch.zeros(4, H, 3, 2, dtype=I32, device=dev)
    calls = {"reserve": lambda: paged.paged_reserve(table, n, count, free, fc, R),
             "slots": lambda: paged.paged_slots(table, n, count, 160, P, R),
             "release": lambda: paged.paged_release(table, n, free, fc, R),
             "bounds": lambda: paged.paged_bounds(kp, table, n, bnd, bs, scales=scales),
             "bounds of part": lambda: paged.paged_bounds(kp, table, n, bnd, bs, n - 1, 9, scales),
             "select": lambda: paged.paged_select(q, bnd, bs, table, n, R, 5),
             "attn": lambda: paged.paged_sparse_attention(q, kp, vp, table, n, index, scales=scales),
             "attn into out": lambda: paged.paged_sparse_attention(q, kp, vp, table, n, index, 0.3, out, scales)}
    if not eight:
        calls["append_slots"] = lambda: paged.paged_append_packed(kp, vp, table, n, count, x, x, slots, starts)
        return calls
    more = torch.ones(4, H, 2, D, device=dev)
    calls.update({"attn of all pages": lambda: paged.paged_attention(q.float(), kp, vp, table, n, scales=scales),
                  "append": lambda: paged.paged_append(kp, vp, table, n, more, more, scales=scales),
                  "append with counts": lambda: paged.paged_append(kp, vp, table, n, more, more, count, scales),
                  "gather": lambda: paged.paged_gather(kp, vp, table, n, 33, scales=scales),
                  "gather in fp32": lambda: paged.paged_gather(kp, vp, table, n, 33, scales, F32)})
    return calls


@pytest.mark.parametrize("code", [BF, F32, E4, I8], ids=["bf16", "fp32", "e4m3", "int8"])
def test_module_makes_the_calls(dev, monkeypatch, code):
    import tabicl_mi355_native as nat
    nat.load()
    real, seen = nat.DIRECT, []

    class Recorder:
        def __getattr__(self, name):
            def call(*a):
                r = getattr(real, name)(*a)
                seen.append((name, r is not None))
                return r
            return call

    calls = _calls(dev, code)
    monkeypatch.setattr(nat, "DIRECT", Recorder())
    for what, call in calls.items():
        seen.clear()
        call()
        torch.cuda.synchronize()
        assert seen == [(what.split()[0], True)], (what, seen)


def test_other_threads_run_meanwhile(dev, tmp_path):
    # stand-ins for the library's functions that sleep without the interpreter: a thread counts on all the while
    import tabicl_mi355_native as nat
    lib = nat.load()
    src, so = tmp_path / "sleep.c", tmp_path / "sleep.so"
    src.write_text("#include <unistd.h>\nlong none(void) { return 0; }\nint pause_(void) { usleep(200000); return 0; }\n")
    subprocess.run(["gcc", "-shared", "-fPIC", str(src), "-o", str(so)], check=True)
    fake = ctypes.CDLL(str(so))
    at = {f: ctypes.cast(getattr(fake, f), ctypes.c_void_p).value for f in ("none", "pause_")}
    calls = {**_calls(dev, BF), **_calls(dev, I8)}
    for call in calls.values():  # whatever is built on a first call
        call()
    torch.cuda.synchronize()
    ticks, stop = [0], threading.Event()

    def count():
        while not stop.is_set():
            ticks[0] += 1
            time.sleep(0.002)

    thread = threading.Thread(target=count)
    try:
        nat.DIRECT.bind({name: at["none" if name.endswith("_bytes") else "pause_"] for name in nat.SIGNATURES})
        thread.start()
        for what, call in calls.items():
            before, t0 = ticks[0], time.monotonic()
            call()
            took = time.monotonic() - t0
            assert took >= 0.2, (what, took)
            assert ticks[0] - before >= 5, what
    finally:
        stop.set()
        nat._bind_direct(lib)
        if thread.is_alive():
            thread.join()
    for call in calls.values():
        call()
    torch.cuda.synchronize()
