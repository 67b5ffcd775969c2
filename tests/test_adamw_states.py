"""States and gradients that do not belong to an optimizer's tensors (ops/adamw.py)."""

import pytest

torch = pytest.importorskip("torch")

from network_operator_amd.ops import adamw  # noqa: E402


@pytest.mark.gpu
@pytest.mark.parametrize("bits", [8, 32])
def test_states_of_other_sizes_are_refused(cuda_device, bits):
    def opt(*sizes):
        return adamw.AdamW([torch.zeros(n, device=cuda_device) for n in sizes], lr=1e-3, state_bits=bits)

    state = opt(256, 512).state_dict()
    for sizes in [(512, 256), (768,), (250, 512), (256, 511), (256, 256, 256), (256, 0, 512)]:
        with pytest.raises(ValueError, match="sizes"):
            opt(*sizes).load_state_dict(state)
    other = opt(256, 512)
    other.load_state_dict(state)
    other.load_state_dict({k: t for k, t in state.items() if k != "sizes"})  # of a state that was kept without them
