import os
import sys
from pathlib import Path

import pytest

ROOT = Path(__file__).resolve().parent.parent
sys.path.insert(0, str(ROOT))


def pytest_configure(config):
    config.addinivalue_line("markers", "gpu: needs a real MI355X (run on the GPU box with -m gpu)")
    config.addinivalue_line("markers", "netns: needs root / user namespaces + AF_PACKET (veth harness)")
    config.addinivalue_line("markers", "slow: long-running")


def _netns_ok():
    try:
        from network_operator_amd.testing import netns

        return netns.available()
    except Exception as e:  # pragma: no cover
        return False, str(e)


# What these test on the node itself is its scale-out NICs (discovery, their place in RCCL's topology).
NEEDS_NICS = {"test_agent_dry_run_on_this_node", "test_node_report_on_this_node", "test_topo_tool_on_this_node",
              "test_require_rdma_dry_run_on_this_node_names_every_rail_without_an_rdma_device",
              "test_fabric_validation_single_gpu", "test_rccl_loads_generated_topology",
              "test_bench_measures_with_the_agents_file_and_reads_rccl_dump"}


def pytest_collection_modifyitems(config, items):
    from network_operator_amd.parallel.fabric_artifacts import pci_netdevs

    ok, why = None, None
    without_nics = not pci_netdevs(os.environ.get("SYSFS_ROOT", "/sys"))
    for item in items:
        if without_nics and item.name in NEEDS_NICS:
            item.add_marker(pytest.mark.skip(reason="this node has no NIC: no netdev is a PCI network function"))
        if "netns" in item.keywords:
            if ok is None:
                ok, why = _netns_ok()
            if not ok:
                item.add_marker(pytest.mark.skip(reason=f"netns harness unavailable: {why}"))


@pytest.fixture(scope="session")
def native():
    from network_operator_amd.agent import native as _n

    return _n()


@pytest.fixture(scope="session")
def cuda_device():
    import torch

    if not torch.cuda.is_available():
        pytest.fail("GPU test selected but no GPU is visible")
    return torch.device("cuda", 0)


@pytest.fixture(scope="session")
def single_rank_pg(cuda_device):
    """A 1-rank RCCL process group for the whole GPU session (one init per process)."""
    import torch.distributed as dist

    import tempfile

    store = os.path.join(tempfile.mkdtemp(prefix="netop-pg-"), "store")  # a FileStore: no TCP port to collide on
    if not dist.is_initialized():
        dist.init_process_group("nccl", init_method=f"file://{store}", rank=0, world_size=1, device_id=cuda_device)
    yield
    if dist.is_initialized():
        dist.destroy_process_group()
