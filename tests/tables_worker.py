"""Child process of test_decode_limits_gpu.py: block tables of 3059 to 3073 requests (16 bytes of shared memory each) as the first calls
of a process, then of the most that a call takes."""
import sys
from pathlib import Path

ROOT = Path(__file__).resolve().parents[1]
sys.path[:0] = [str(ROOT), str(ROOT / "softhier-mlir_b200"), str(ROOT / "tests")]

import numpy as np  # noqa: E402

from oracle import decode as D  # noqa: E402
from softhier_cuda.runtime import Runtime  # noqa: E402
from test_decode_gpu import _run_tables, _tables_case  # noqa: E402


def main(many: bool) -> None:
    rt = Runtime.open(0, arena_bytes=1 << 20)
    for R in (3059, 3060, 3064, 3071, 3073, 8192):
        rng = np.random.default_rng(R)
        lens, add = rng.integers(0, 100, R), rng.integers(0, 60 if many else 2, R)
        lens, add, table, ring, pool = _tables_case(lens, add, 16, 12, 12 * R, R)
        t_cap = int(add.sum()) + (80000 if many else 9)          # four tokens per thread, or one
        want = D.kv_tables(lens, add, 16, table, ring, pool, t_cap)
        got = _run_tables(rt, lens, add, 16, table, ring, pool, t_cap, True)
        for i, (w, x) in enumerate(zip(want, got)):
            np.testing.assert_array_equal(x[:3] if i == 2 else x, w)
    print("OK")


if __name__ == "__main__":
    main(sys.argv[1] == "many")
