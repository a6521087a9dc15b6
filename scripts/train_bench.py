"""GPU time of the training operators' C entries (lbm_hip_norm_forward / _backward, lbm_hip_dropout) on prepared descriptors.  The operands
rotate over copies (1.5 GB in all) so that nothing is found in a cache.  usage: python scripts/train_bench.py [rows cols [x_type [residual_type]]]
without arguments: the tracker's sizes, wide rows, rows of odd length, dropout."""
import ctypes as C
import os
import sys

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))
import torch
from lbm_amd import hip

lib = hip.load()
TYPES = {"f32": (torch.float32, 0), "f16": (torch.float16, 1), "bf16": (torch.bfloat16, 2)}


def time_us(calls, repeats=7):
    stream = torch.cuda.current_stream().cuda_stream
    for f in calls:
        f(stream)
    out = []
    for _ in range(repeats):
        a, b = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
        a.record()
        for f in calls:
            f(stream)
        b.record()
        torch.cuda.synchronize()
        out.append(a.elapsed_time(b) * 1e3 / len(calls))
    return sorted(out)[len(out) // 2]


def ptr(t):
    return None if t is None else t.data_ptr()


def norm(rows, cols, x="f32", res=None):
    (tx, cx), (tr, cr) = TYPES[x], TYPES[res or x]
    copies = max(1, min(12, int(1.5e9 / (rows * cols * (2 * tx.itemsize + 3 * tr.itemsize)))))
    forward, backward, keep = [], [], []
    for _ in range(copies):
        X = torch.randn(rows, cols, device="cuda").to(tx)
        R = torch.randn(rows, cols, device="cuda").to(tr) if res else None
        W, B = torch.ones(cols, device="cuda"), torch.zeros(cols, device="cuda")
        DY = torch.randn(rows, cols, device="cuda").to(tr)
        Y, DX, DR, S, DW, DB = torch.empty_like(DY), torch.empty_like(X), torch.empty_like(DY) if res else None, torch.empty(2, rows, device="cuda"), \
            torch.empty_like(W), torch.empty_like(B)
        n = lib.lbm_hip_norm_workspace_bytes(rows, cols)
        ws = torch.empty(n, device="cuda", dtype=torch.uint8)
        d = hip.NormDesc(ptr(X), ptr(R), ptr(W), ptr(B), ptr(Y), ptr(S), ptr(S) + 4 * rows, ptr(DY), ptr(DX), ptr(DR), ptr(DW), ptr(DB), ptr(ws), n,
                         rows, cols, cols, cols, cols, cx, cr, 0, 1e-5, 0.1 if res else 0.0, 123, 4, None)
        keep.append((X, R, W, B, DY, Y, DX, DR, S, DW, DB, ws, d))
        forward.append(lambda s, d=d: hip._check(lib.lbm_hip_norm_forward(C.byref(d), s), "forward"))
        backward.append(lambda s, d=d: hip._check(lib.lbm_hip_norm_backward(C.byref(d), s), "backward"))
    rep, n = max(1, 20 // copies), rows * cols
    f, b = time_us(forward * rep), time_us(backward * rep)
    fb, bb = n * (tx.itemsize + tr.itemsize * (2 if res else 1)), n * (2 * tx.itemsize + tr.itemsize * (3 if res else 1))
    print("%-11s %8d x %-6d forward %8.2f us %5.2f TB/s   backward %8.2f us %5.2f TB/s" % (x + ("+" + res if res else ""), rows, cols, f, fb / f / 1e6, b, bb / b / 1e6), flush=True)


def drop(n, x):
    t, code = TYPES[x]
    copies = max(1, min(12, int(1.5e9 / (2 * n * t.itemsize))))
    calls, keep = [], []
    for _ in range(copies):
        X = torch.randn(n, device="cuda").to(t)
        Y = torch.empty_like(X)
        keep.append((X, Y))
        calls.append(lambda s, X=X, Y=Y: hip._check(lib.lbm_hip_dropout(ptr(X), ptr(Y), n, code, 0.1, 123, None, 4, s), "dropout"))
    us = time_us(calls * max(1, 20 // copies))
    print("dropout %-4s %12d %8.2f us %5.2f TB/s" % (x, n, us, 2 * n * t.itemsize / us / 1e6), flush=True)


if __name__ == "__main__":
    if len(sys.argv) > 2:
        norm(int(sys.argv[1]), int(sys.argv[2]), *sys.argv[3:])
    else:
        for a in [(8, 256), (1024, 256), (65536, 256, "f16"), (589824, 256, "bf16"), (589824, 256, "f32"), (16320, 257, "bf16"), (146914, 1021, "f16"), (8192, 8192, "bf16"),
                  (9000, 16384, "bf16"), (8000, 20000, "bf16"), (64, 256, "f32", "f32"), (9216, 256, "f16", "f32"), (4099, 1537, "bf16", "bf16"), (589824, 256, "bf16", "bf16"),
                  (589824, 256, "f32", "f32"), (589824, 256, "f16", "f32"), (589824, 256, "bf16", "f32"), (150000, 1024, "bf16", "bf16"), (148000, 1021, "f16", "f16"),
                  (36000, 4096, "bf16", "bf16"), (18000, 8192, "bf16", "bf16"), (9000, 16384, "bf16", "bf16"), (9000, 16384, "f16", "f32"), (8000, 20000, "bf16", "bf16")]:
            norm(*a)
        for a in [(1 << 20, "f32"), (9217 * 1021, "f16"), (65536 * 1024, "bf16"), (589824 * 256, "f32"), (589824 * 256, "bf16")]:
            drop(*a)
