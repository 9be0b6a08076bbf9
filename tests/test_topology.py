"""utils/topology.py on machines without xGMI links."""
import pytest

from vodascheduler_amd.utils.topology import from_dump

CPU = "== /nodes/0/properties\ncpu_cores_count 64\nsimd_count 0\n"
PCIE = "== /nodes/{0}/io_links/0/properties\ntype 2\nnode_from {0}\nnode_to 0\nweight 20\n"


@pytest.mark.parametrize("gpus", [0, 1, 2])
def test_gpus_without_xgmi(gpus):
    t = from_dump(CPU + "".join(f"== /nodes/{i}/properties\nsimd_count 1024\n" + PCIE.format(i) for i in range(1, gpus + 1)))
    assert t.n == gpus and t.links_per_gpu() == 0 and not t.xgmi
    assert t.numa == {i: 0 for i in range(gpus)}
    assert t.full_mesh() == (gpus == 1)
    assert t.bucket_mb(8) >= 32
