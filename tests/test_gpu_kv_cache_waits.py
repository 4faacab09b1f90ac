"""The waits of the cache attention's tensor-core kernel, in the second build of the library (lib/waittest: a wait budget of about a
millisecond, and hooks that make tiles or rows late or leave a tile out).  Tiles and rows that come late change no bit of the result: whoever
depends on one waits for it.  A tile that never comes ends the launch in order: the host reads AR_ERR_DEVICE_WAIT, later CTAs
leave at once, and the next launch on the same GPU gives the bits of the launch before.  In a child process, so that the
two libraries never meet in one address space."""
from __future__ import annotations

import subprocess
import sys
import textwrap
from pathlib import Path

import pytest

pytestmark = pytest.mark.gpu

ROOT = Path(__file__).resolve().parent.parent

CHILD = textwrap.dedent('''
    import sys, time
    from pathlib import Path
    sys.path.insert(0, sys.argv[1])
    import torch
    from autorust_b200 import _abi
    _abi.LIB_DIR = Path(sys.argv[1]) / "autorust_b200" / "lib" / "waittest"
    from autorust_b200 import ops
    L = _abi.load()
    g = torch.Generator(device="cuda").manual_seed(0)
    rand = lambda *s: torch.randn(s, device="cuda", generator=g).to(torch.bfloat16)
    ints = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")
    B, heads = 3, 4
    for D, page, n, m in ((128, 64, 700, 700), (64, 16, 700, 700), (128, 32, 3000, 200)):  # (the last in parts)
        pages = -(-n // page)
        cache = ops.kv_cache(B * pages, heads, page, D)
        table = torch.randperm(B * pages, device="cuda", generator=g).to(torch.int32).view(B, pages)
        lengths, starts = ints([n, 129, 300]), ints([0, n, n + 129, n + 429])
        few = ints([0, m, m + 29, m + 49])
        # rows whose maximum keeps growing: the accumulators are rescaled at many steps
        grow = torch.linspace(0.2, 3.0, n, device="cuda")[:, None, None]
        k = rand(n + 429, heads, D)
        k[:n] = (k[:n].float() * grow).to(torch.bfloat16)
        ops.kv_cache_append(cache, k, rand(n + 429, heads, D), table, lengths, starts)
        q = rand(m + 49, 2 * heads, D)
        run = lambda: ops.kv_cache_attention(cache, q, table, lengths, few)
        want = run()
        assert ops.last_status(None) == _abi.AR_OK
        for late in ((5000, 0, 0), (0, 5000, 0), (3000, 3000, 0), (20000, 1000, 0), (0, 0, 5000), (0, 0, 20000)):
            assert L.ar_test_late_cache_tiles(*late) == 0
            assert torch.equal(run(), want), late
            assert ops.last_status(None) == _abi.AR_OK
        assert L.ar_test_late_cache_tiles(0, 0, 0) == 0
        for tile in (0, 1):
            assert L.ar_test_skip_cache_tile(tile) == 0
            t0 = time.perf_counter()
            run()
            torch.cuda.synchronize()
            assert time.perf_counter() - t0 < 1.0
            assert ops.last_status(None) == _abi.AR_ERR_DEVICE_WAIT and ops.last_status(None) == _abi.AR_OK
            assert L.ar_test_skip_cache_tile(-1) == 0
            assert torch.equal(run(), want) and ops.last_status(None) == _abi.AR_OK
    print("done")
''')


def test_late_and_missing_tiles(attn_lib):
    out = subprocess.run([sys.executable, "-c", CHILD, str(ROOT)], capture_output=True, text=True, timeout=300)
    assert out.returncode == 0 and "done" in out.stdout, out.stdout + out.stderr
