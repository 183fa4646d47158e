"""Workspace of the entries beside the products over the sizes that they accept, on the host (tests/host_runtime.py: no kernel runs)."""
from tests import host_runtime


def test_workspace_of_the_adapters(tmp_path_factory):
    """Sums over the rank of every row (each split of the columns has its own: splits times slots of 64 rows are no more than 512 and a round of slots), again added up where dx and
    dA both want them, and up to 128 MiB of the gradients' parts; a call that needs no more than 128 MiB stays within a stream's own block."""
    host_runtime.run(tmp_path_factory, """
import random
P, MIB = 1 << 40, 1 << 20
rng = random.Random(5)
runtime.host_budget(1 << 62)
above = 0
for _ in range(600):
    rows, adapters, rank = int(2 ** rng.uniform(0, 21)), int(2 ** rng.uniform(0, 12)), rng.randint(1, 128)
    k, n = int(2 ** rng.uniform(3, 15)), int(2 ** rng.uniform(3, 15))
    pitch = (rank + 15) // 16 * 16
    sums = 4 * pitch * min(16 * rows, 64 * 512 + 2 * rows + 64)
    for call, most in ((lambda: lib.qgemm_add_adapters(BF16, BF16, P, n, P, k, P, P, P, P, 2 * P, n, P, rows, adapters, rank, k, n, 0), sums),
                       (lambda: lib.qgemm_add_adapters_backward(BF16, BF16, F32, P, n, P, k, P, P, P, P, P, P, k, 2 * P, k, P, P, rows, adapters, rank, k, n, 0),
                        sums + 4 * rank * rows + 128 * MIB + 4096)):
        lib.qgemm_shutdown()
        events()
        assert call() == 0
        took = [int(e.split()[1]) for e in events() if e.startswith("malloc")]
        above += max(took, default=0) > 128 * MIB
        assert max(took, default=0) <= max(128 * MIB, most), (rows, adapters, rank, k, n, took, most)
assert above                                               # (some of these need more: then it is the shared block's)
""")
