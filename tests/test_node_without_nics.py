"""Which netdevs count as a node's NICs where tests and smoke() ask whether it has any."""

from network_operator_amd.parallel.fabric_artifacts import pci_netdevs


def test_pci_netdevs(tmp_path):
    assert pci_netdevs(str(tmp_path)) == []  # no class/net at all
    net = tmp_path / "class" / "net"
    (net / "lo").mkdir(parents=True)  # no device
    (net / "eth0" / "device").mkdir(parents=True)  # a virtio device: its PCI function is one above
    (net / "eth0" / "device" / "vendor").write_text("0x1af4\n")
    assert pci_netdevs(str(tmp_path)) == []
    for name, cls in (("ens1", "0x020000\n"), ("ib0", "0x020700\n"), ("odd", "0x030000\n")):
        dev = tmp_path / "devices" / name
        dev.mkdir(parents=True)
        (dev / "class").write_text(cls)
        (net / name).mkdir()
        (net / name / "device").symlink_to(dev)
    assert pci_netdevs(str(tmp_path)) == ["ens1", "ib0"]
