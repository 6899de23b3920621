"""The 8-bit operators' checks of their arguments and the block matrix's layouts (no GPU)."""
import pytest
import torch

from yoda_scheduler_amd.ops import fp8
from yoda_scheduler_amd.ops.fp8 import BLOCK, E4M3, E8M0, BlockMatrix


def _matrix(rows, cols, block_rows=1, scale_dtype=torch.float32):
    kb = fp8.blocks(cols)
    return BlockMatrix(torch.zeros(rows, kb * BLOCK).to(E4M3),
                       torch.ones(rows if block_rows == 1 else fp8.blocks(rows), kb).to(scale_dtype), cols, block_rows)


def test_unpadded_values_are_padded_with_zeros_and_scales_laid_out():
    v = torch.arange(3 * 130, dtype=torch.float32).view(3, 130).fmod(9).to(E4M3)
    s = torch.tensor([[1.0, 2.0], [3.0, 4.0], [5.0, 6.0]])
    m = BlockMatrix(v, s)
    assert m.shape == (3, 130) and m.data.shape == (3, 256) and m.values.shape == (3, 130)
    assert torch.equal(m.values.float(), v.float())
    assert torch.equal(m.data[:, 130:].float(), torch.zeros(3, 126))
    assert m.scales.stride() == (1, 8) and torch.equal(m.scales, s)
    w = BlockMatrix(v, torch.tensor([[2.0, 0.5]]).to(E8M0), block_rows=128)
    assert w.scales.is_contiguous() and w.scales.shape == (1, 2)
    assert "3x130" in repr(w)


def test_padded_values_are_taken_as_they_are():
    v = torch.zeros(16, 256).to(E4M3)
    s = torch.ones(2, 16).t()
    m = BlockMatrix(v, s, cols=200)
    assert m.data.data_ptr() == v.data_ptr() and m.scales.data_ptr() == s.data_ptr() and m.cols == 200


@pytest.mark.parametrize("values,scales,kw,error", [
    (torch.zeros(4, 128), torch.ones(4, 1), {}, TypeError),                                   # not e4m3
    (torch.zeros(128).to(E4M3), torch.ones(1, 1), {}, TypeError),                             # one axis
    (torch.zeros(4, 128).to(E4M3), torch.ones(4, 1, dtype=torch.float64), {}, TypeError),     # scales' type
    (torch.zeros(4, 128).to(E4M3), torch.ones(4), {}, TypeError),
    (torch.zeros(4, 128).to(E4M3), torch.ones(4, 2), {}, ValueError),                         # scales' shape
    (torch.zeros(4, 128).to(E4M3), torch.ones(4, 1), {"block_rows": 128}, ValueError),
    (torch.zeros(4, 128).to(E4M3), torch.ones(4, 1), {"block_rows": 64}, ValueError),
    (torch.zeros(4, 256).to(E4M3), torch.ones(4, 1), {"cols": 100}, ValueError),              # padded too far
    (torch.zeros(4, 0).to(E4M3), torch.ones(4, 0), {}, ValueError),
    (torch.zeros(4, 128).to(E4M3), torch.ones(4, 1, device="meta"), {}, ValueError),          # another device
])
def test_block_matrix_refuses(values, scales, kw, error):
    with pytest.raises(error):
        BlockMatrix(values, scales, **kw)


@pytest.mark.parametrize("x,kw,error", [
    (torch.zeros(4, 128), {}, ValueError),                                                    # not on a GPU
    (torch.zeros(4, 128, dtype=torch.float64), {}, TypeError),
    (torch.zeros(4, 128, dtype=torch.int8), {}, TypeError),
    (torch.zeros(128), {}, ValueError),
    (torch.zeros(2, 4, 128), {}, ValueError),
    (torch.zeros(128, 4).t(), {}, ValueError),                                                # columns apart
])
def test_quantize_and_norm_refuse(x, kw, error):
    with pytest.raises(error):
        fp8.quantize(x, **kw)
    with pytest.raises(error):
        fp8.add_rms_norm(x, torch.ones(x.shape[-1], dtype=x.dtype), **kw)


def test_scale_dtype_and_gradients_are_refused():
    with pytest.raises(TypeError):
        fp8._scale_kind(torch.float16)
    w = torch.ones(4, requires_grad=True)
    with pytest.raises(RuntimeError):
        fp8._no_grad(None, w)
    with torch.no_grad():
        fp8._no_grad(w)


@pytest.mark.parametrize("a,b,kw,error", [
    (_matrix(4, 128, 128), _matrix(4, 128, 128), {}, ValueError),                             # a's blocks
    (_matrix(4, 128), _matrix(4, 128), {}, ValueError),                                       # b's blocks
    (_matrix(4, 128), _matrix(4, 129, 128), {}, ValueError),                                  # columns
    (_matrix(4, 128), _matrix(4, 128, 128, E8M0), {}, TypeError),                             # two kinds of scales
    (_matrix(4, 128), _matrix(4, 128, 128), {}, ValueError),                                  # not on a GPU
])
def test_matmul_refuses(a, b, kw, error):
    with pytest.raises(error):
        fp8.matmul(a, b, **kw)


def test_what_is_no_plain_tensor_is_refused():
    x = torch.ones(4, 128)
    for bad, error in ((None, TypeError), ([1.0], TypeError), (torch._neg_view(x), ValueError), (x.to_sparse(), ValueError)):
        with pytest.raises(error):
            fp8._refuse_matrix(bad, "x")


def test_scales_that_are_learned_are_refused():
    """A block matrix takes them; a product that would lose their gradient does not."""
    b = fp8.BlockMatrix(torch.zeros(4, 128).to(E4M3), torch.ones(1, 1, requires_grad=True), block_rows=128)
    a = _matrix(4, 128)
    with pytest.raises(RuntimeError, match="backward"):
        fp8.matmul(a, b)
    with torch.no_grad(), pytest.raises(ValueError, match="GPU"):
        fp8.matmul(a, b)


class FakeProber:
    """A node's probes without a GPU: HIP ordinal d is amd-smi index d."""

    def __init__(self, backend, wrong=(), nbytes=1 << 28):
        self.backend, self.wrong, self.nbytes, self.runs = backend, set(wrong), nbytes, []

    def count(self):
        return self.backend.count

    def bus_id(self, d):
        return self.backend._bdf(d)

    def bandwidth_gbps(self, d, nbytes):
        return 6000.0

    def pattern_errors(self, d, nbytes):
        return 0

    def matrix_bytes(self):
        return self.nbytes

    def matrix(self, d):
        self.runs.append(d)
        return (5 if d in self.wrong else 0), 2500.0


def test_matrix_probe_counts_towards_health():
    from yoda_scheduler_amd.sniffer.collector import FakeBackend
    from yoda_scheduler_amd.sniffer.publisher import SnifferAgent
    be = FakeBackend(4, node="n")
    be.tenants[1] = (1, 32)                       # a tenant: not probed
    prober = FakeProber(be, wrong={2})
    agent = SnifferAgent(None, "n", be, probe=True, prober=prober, fail_threshold=2, probe_matrix=True)
    for k in range(2):
        res = agent.run_probes()
    health = {c.id: c.health for c in agent.build().status.card_list}
    assert health == {0: "Healthy", 1: "Healthy", 2: "Unhealthy", 3: "Healthy"}
    assert prober.runs == [0, 2, 3] * 2 and res[2]["matrix_errors"] == 5 and res[2]["pattern_errors"] == 0
    assert agent.measured_tflops == {0: 2500.0, 2: 2500.0, 3: 2500.0}
    prober.wrong.clear()
    agent.run_probes()
    assert {c.health for c in agent.build().status.card_list} == {"Healthy"}


def test_matrix_probe_is_off_by_default_and_keeps_to_its_share_of_memory():
    from yoda_scheduler_amd.sniffer.collector import FakeBackend
    from yoda_scheduler_amd.sniffer.publisher import SnifferAgent
    be = FakeBackend(2, node="n")
    prober = FakeProber(be)
    res = SnifferAgent(None, "n", be, probe=True, prober=prober).run_probes()
    assert not prober.runs and "matrix_errors" not in res[0]
    prober = FakeProber(be, nbytes=(be.spec.hbm_mb // 4 + 1) << 20)
    agent = SnifferAgent(None, "n", be, probe=True, prober=prober, probe_matrix=True)
    res = agent.run_probes()
    assert not prober.runs and res[0]["matrix_skipped"] and res[0]["fail_streak"] == 0
    from yoda_scheduler_amd.cmd.sniffer import build_parser
    assert build_parser().parse_args([]).probe_matrix is False
    assert build_parser().parse_args(["--probe", "--probe-matrix"]).probe_matrix is True


def test_tangents_are_refused():
    """A forward-mode tangent would be lost as a gradient would; under no_grad too, which leaves forward mode on."""
    from torch.autograd import forward_ad
    x = torch.ones(4, 128)
    with forward_ad.dual_level():
        dual = forward_ad.make_dual(x, torch.ones_like(x))
        b = fp8.BlockMatrix(torch.zeros(4, 128).to(E4M3), forward_ad.make_dual(torch.ones(1, 1), torch.ones(1, 1)),
                            block_rows=128)
        for _ in range(2):
            with pytest.raises(RuntimeError, match="forward-mode"):
                fp8._no_grad(None, dual)
            with pytest.raises(RuntimeError, match="forward-mode"):
                fp8.matmul(_matrix(4, 128), b)
            with torch.no_grad(), pytest.raises(RuntimeError, match="forward-mode"):
                fp8._no_grad(dual)
        fp8._no_grad(forward_ad.unpack_dual(dual).primal)
        with torch.inference_mode():
            fp8._no_grad(dual)
    fp8._no_grad(x)


def test_another_torch_makes_the_module_stale(tmp_path, monkeypatch):
    """The module is compiled against torch's C++ internals: its build id names the torch it was built with."""
    from yoda_scheduler_amd.ops import build

    def ids(where, version):
        d = tmp_path / where
        d.mkdir(exist_ok=True)
        (d / "version.py").write_text(f"__version__ = '{version}'\n")
        monkeypatch.setattr(build, "torch_root", lambda: d)
        return build.source_hash("fp8"), build.source_hash("hip")

    here, other, moved = ids("a", "2.10.0"), ids("a", "2.11.0"), ids("b", "2.10.0")
    assert len({here[0], other[0], moved[0]}) == 3 and here[1] == other[1] == moved[1]
    assert ids("a", "2.10.0") == here
    monkeypatch.setattr(build, "torch_root", lambda: None)
    assert build.source_hash("fp8") not in (here[0], other[0], moved[0])
