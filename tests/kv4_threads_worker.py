"""First calls of a process into the 4-bit operators, from several threads at once (started by ``tests/test_gpu_kv4.py``)."""

import os
import sys
import threading

import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))
from daser_b200.ops import _lib, attention, kv_ops  # noqa: E402

THREADS, CTX = 8, 500


def main() -> int:
    pool = kv_ops.PagedKV4Pool.zeros(1, 64, 1, "cuda")
    bounds = kv_ops.PageBounds.for_pool(pool)
    i32 = dict(dtype=torch.int32, device="cuda")
    table, ctx = torch.arange(64, **i32)[None], torch.tensor([CTX], **i32)
    for name in _lib._KV4_ARGS:
        _lib.kv4_fn(name)  # symbols are looked up before the threads start: they meet inside the entry points
    gate, errors = threading.Barrier(THREADS), []

    def work(i: int) -> None:
        try:
            n = 16 if i % 2 else 1
            q = torch.zeros(n, 8, 128, dtype=torch.bfloat16, device="cuda")
            out, start = torch.full_like(q, 7.0), torch.tensor([0, n], **i32)
            torch.cuda.synchronize()
            with torch.cuda.stream(torch.cuda.Stream()):
                gate.wait()
                attention.paged_attention(q, out, pool, 0, table, start, ctx, n, CTX, 1, 1.0, None, nsplit=None)
                gate.wait()
                pages = attention.select_pages(q, bounds, 0, table, start, ctx, n, CTX, 8)
                gate.wait()
                attention.sparse_paged_attention(q, out, pool, 0, table, start, ctx, pages, n, 1.0)
            torch.cuda.synchronize()
            if out.any():
                raise RuntimeError("a pool of zeros gave something else")
        except Exception as exc:  # noqa: BLE001
            errors.append(repr(exc))
            gate.abort()

    threads = [threading.Thread(target=work, args=(i,)) for i in range(THREADS)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    print(errors or "ok")
    return 1 if errors else 0


if __name__ == "__main__":
    sys.exit(main())
