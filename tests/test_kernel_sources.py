"""Rules of the CUDA programming model that a run cannot show to be broken, read off the kernel sources."""
import re
from pathlib import Path

import pytest

CSRC = Path(__file__).parents[1] / "param_decomp_b200" / "ops" / "csrc"


def _kernels(path: Path) -> dict[str, str]:
    parts = re.split(r"(?=__global__)", path.read_text())[1:]
    return {re.search(r"(\w+_kernel)\(", p).group(1): p for p in parts}


@pytest.mark.parametrize("source", sorted(p.name for p in CSRC.glob("*.cu")))
def test_cluster_barrier_before_a_peers_shared_memory(source):
    """A CTA of a cluster may touch another one's shared memory only once that one is known to run: a cluster barrier stands
    before the first address mapped to a peer."""
    for name, body in _kernels(CSRC / source).items():
        mapped, barrier = body.find("mapa_shared("), body.find("cluster_sync_all()")
        assert mapped < 0 or 0 <= barrier < mapped, name


def test_generic_stores_into_bulk_copy_targets_are_fenced():
    """vocab_kl writes over the columns past V in a buffer that the next row's bulk copy overwrites: the writing thread's
    proxy fence follows each such store."""
    body = _kernels(CSRC / "vocab_kl.cu")["vocab_kl_rows_kernel"]
    stores = [m.end() for m in re.finditer(r"ta\[k\] = tb\[k\] = [^;]*;", body)]
    assert stores and all("fence_proxy_async_smem();" in body[at : at + 60] for at in stores)


def test_a_clusters_end_is_handed_over_like_its_rows():
    """top_logits: what a block's selecting warps read of a row is written again two rows on. A block knows that they have read it
    from the cluster's meeting in every row; behind the last one, before the end marker, the cluster meets once more."""
    body = _kernels(CSRC / "top_logits.cu")["top_logits_kernel"]
    rows, end = body.index("for (int r = blockIdx.x / cs"), body.index("sh.work[n & 1].row = -1")
    behind = body[body.index("r = next;", rows) : end]
    meeting = re.search(r"wait_pair\(selected, n - 2\).*mbar_arrive_cluster\(mapa_shared\(met, lane\)\).*short_wait<true>\(met, n & 1", behind, re.S)
    assert meeting, "no meeting between the last row and the end marker"
