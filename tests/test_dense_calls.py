"""The dense operators' calls without a GPU, over the stand-in for the HIP runtime: streams, arrays and what is refused."""

from pathlib import Path

from .fake_runtime import run_fake
from .test_dense import PRELUDE


def test_per_thread_streams(tmp_path: Path) -> None:
    """hipStreamPerThread (2) names another stream in each thread: a call on it waits for the workspace's last one, whichever
    thread that came from."""
    run_fake(tmp_path, PRELUDE + """
l = linear(4096, 1024)
x, y = arr(300, 1024), arr(300, 4096)
l(x, y, stream=2)
before = hip.waits
l(x, y, stream=2)
assert hip.waits == before + 1
l(x, y, stream=5); l(x, y, stream=5)
assert hip.waits == before + 2
""")
