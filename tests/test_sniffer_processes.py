"""Who holds a GPU, where the driver's process list cannot be read, what the probes make of it, and their own process."""
import os
import signal
import subprocess
import sys

import pytest

from yoda_scheduler_amd.sniffer.collector import FakeBackend, samples_to_scv
from yoda_scheduler_amd.sniffer.publisher import SnifferAgent


class Prober:
    def __init__(self, backend):
        self.backend, self.probed = backend, []

    def count(self):
        return self.backend.count

    def bus_id(self, d):
        return self.backend._bdf(d)

    def bandwidth_gbps(self, d, nbytes):
        self.probed.append(d)
        return 6000.0

    def pattern_errors(self, d, nbytes):
        return 0

    def matrix_bytes(self):
        return 1 << 28

    def matrix(self, d):
        return 0, 2500.0


def test_holders_are_found_by_their_open_files(tmp_path):
    from yoda_scheduler_amd.ops.native import load_native
    mod = load_native("sniffer", "yoda_scheduler_amd._native._yoda_sniffer")

    def process(pid, *files):
        d = tmp_path / str(pid) / "fd"
        d.mkdir(parents=True)
        for i, f in enumerate(files):
            os.symlink(f, d / str(i))

    process(10, "/dev/null", "/dev/kfd", "/dev/dri/renderD128")
    process(11, "/dev/kfd", "/dev/dri/renderD128", "/dev/dri/renderD129", "/dev/dri/renderD129")
    process(12, "/dev/dri/renderD130")                             # a display, no compute
    process(13, "/dev/kfd")
    process(14, "anon_inode:[eventfd]", "/dev/dri/card0" + "x" * 80)
    (tmp_path / "15").mkdir()                                       # cannot be looked into
    (tmp_path / "self").mkdir()
    assert mod.kfd_holders(str(tmp_path)) == {128: 2, 129: 1}
    assert mod.kfd_holders(str(tmp_path / "none")) == {}
    assert isinstance(mod.kfd_holders(), dict)


@pytest.mark.parametrize("matrix", [False, True])
def test_a_gpu_whose_processes_are_unknown_is_not_probed(matrix):
    be = FakeBackend(3, node="n")
    prober = Prober(be)
    agent = SnifferAgent(None, "n", be, probe=True, prober=prober, probe_matrix=matrix)
    s = be.sample()
    s[0]["processes"] = -1
    del s[1]["processes"]
    res = agent.run_probes(s)
    assert prober.probed == [2] and "unknown" in res[0]["skipped"] and "unknown" in res[1]["skipped"]
    assert set(agent.probe_skipped) == {0, 1} and 0 not in agent.probe_fail_streak
    agent.run_probes()                                              # known again
    assert prober.probed == [2, 0, 1, 2] and not agent.probe_skipped


def test_occupancy_is_not_taken_from_a_list_that_could_not_be_read():
    s = FakeBackend(2, node="n").sample()
    for x in s:
        x |= {"processes": 2, "processCUs": 0, "gfxActivity": 70, "errors": ["process_list"]}
    card = samples_to_scv("n", s).status.card_list[0]
    assert card.processes == 2 and card.occupancy_source == "gfx-activity" and card.cu_occupancy == 70.0


def _alone(code):
    """Run in a process that has loaded nothing yet."""
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    r = subprocess.run([sys.executable, "-c", code], cwd=root, capture_output=True, text=True, timeout=100)
    assert r.returncode == 0, r.stderr[-2000:]
    return r.stdout


def test_the_agent_keeps_no_context_of_its_own():
    """Probes run in a process that ends: the agent's own would be on every card from the first probe on, so that the
    next sample finds them all busy."""
    out = _alone("from yoda_scheduler_amd.sniffer.publisher import HipProber\n"
                 "p = HipProber(); print(p.matrix_bytes()); p.close()\n"
                 "print('libamdhip64' in open('/proc/self/maps').read())")
    size, mapped = out.split()
    assert int(size) > 1 << 27 and mapped == "False"


def test_a_probing_process_that_fails_hangs_or_ends(monkeypatch):
    from yoda_scheduler_amd.sniffer import probe
    w = probe.Worker(timeout=60)
    with pytest.raises(probe.ProbeError, match="KeyError"):
        w.ask("nothing of the kind")
    first = w._child.pid
    assert w.ask("matrix_bytes") > 0 and w._child.pid == first         # an error is an answer
    w._child.kill()
    with pytest.raises(probe.ProbeError, match="ended .status -9"):
        w.ask("matrix_bytes")
    assert w.ask("matrix_bytes") > 0 and w._child.pid != first         # and the next question has a new process
    w.timeout = 0.5
    os.kill(w._child.pid, signal.SIGSTOP)
    with pytest.raises(probe.ProbeError, match="no answer in 0.5 s"):
        w.ask("matrix_bytes")
    w.close()
    w.close()


@pytest.mark.gpu
def test_probes_leave_no_context_behind(require_gpu):
    out = _alone("import os\n"
                 "from yoda_scheduler_amd.sniffer.publisher import HipProber\n"
                 "p = HipProber()\n"
                 "print(p.count(), p.bus_id(0), p.bandwidth_gbps(0, 64 << 20) > 100, p.pattern_errors(0, 64 << 20), p.matrix(0)[0])\n"
                 "p.close()\n"
                 "links = [os.readlink(f'/proc/self/fd/{f}') for f in os.listdir('/proc/self/fd') if os.path.lexists(f'/proc/self/fd/{f}')]\n"
                 "print(any('kfd' in x or 'renderD' in x for x in links))")
    first, second = out.split("\n")[:2]
    assert first.split()[0] == "1" and first.split()[2:] == ["True", "0", "0"] and second == "False", out


class FailingProber(Prober):
    """Probes of some cards raise, others find errors."""

    def __init__(self, backend, **fails):
        super().__init__(backend)
        self.fails = fails                    # what: {card: what it raises or returns}

    def _or(self, what, d, value):
        v = self.fails.get(what, {}).get(d, value)
        if isinstance(v, Exception):
            raise v
        return v

    def bandwidth_gbps(self, d, nbytes):
        self.probed.append(d)
        return self._or("bandwidth", d, 6000.0)

    def pattern_errors(self, d, nbytes):
        return self._or("pattern", d, 0)

    def matrix(self, d):
        return self._or("matrix", d, (0, 2500.0))


def test_a_probe_that_raises_is_a_failed_one_and_the_rest_counts():
    be = FakeBackend(4, node="n")
    prober = FailingProber(be, matrix={0: RuntimeError("hipError 700"), 2: RuntimeError("")}, pattern={0: 7, 1: 9},
                           bandwidth={3: RuntimeError("no memory")})
    agent = SnifferAgent(None, "n", be, probe=True, prober=prober, fail_threshold=2, probe_matrix=True)
    for k in range(2):
        res = agent.run_probes()
    assert prober.probed == [0, 1, 2, 3] * 2
    assert res[0]["pattern_errors"] == 7 and "700" in res[0]["error"] and res[2]["error"] and "no memory" in res[3]["error"]
    assert [res[i]["fail_streak"] for i in range(4)] == [2] * 4
    assert {c.health for c in agent.build().status.card_list} == {"Unhealthy"}
    assert set(agent.measured_bw) == {0, 1, 2} and set(agent.measured_tflops) == {1}
    prober.fails.clear()
    agent.run_probes()
    assert {c.health for c in agent.build().status.card_list} == {"Healthy"}


def test_a_skipped_matrix_check_clears_no_card_that_it_failed():
    be = FakeBackend(2, node="n")
    prober = FailingProber(be, matrix={0: (3, 2500.0)}, pattern={1: 4})
    agent = SnifferAgent(None, "n", be, probe=True, prober=prober, fail_threshold=2, probe_matrix=True)
    agent.run_probes()
    agent.run_probes()
    assert {c.health for c in agent.build().status.card_list} == {"Unhealthy"}
    prober.fails.clear()
    prober.matrix_bytes = lambda: 1 << 50                           # no room: not repeated
    res = agent.run_probes()
    assert res[0]["matrix_skipped"] and res[0]["fail_streak"] == 2 and res[1]["fail_streak"] == 0
    assert [c.health for c in agent.build().status.card_list] == ["Unhealthy", "Healthy"]
    prober.fails["pattern"] = {0: 1}
    assert agent.run_probes()[0]["fail_streak"] == 3
    prober.fails.clear()
    assert agent.run_probes()[0]["fail_streak"] == 3
    del prober.matrix_bytes
    assert agent.run_probes()[0]["fail_streak"] == 0
    assert {c.health for c in agent.build().status.card_list} == {"Healthy"}
    # one that raised is a matrix failure as well
    prober.fails["matrix"] = {1: RuntimeError("hipError 700")}
    agent.run_probes()
    prober.matrix_bytes = lambda: 1 << 50
    assert agent.run_probes()[1]["fail_streak"] == 1


def test_an_error_of_the_runtime_ends_the_probing_process(monkeypatch):
    """One card's fault can stay with the process; the next card's probes are not to meet it."""
    from yoda_scheduler_amd.sniffer import probe
    w = probe.Worker(timeout=60)
    with pytest.raises(probe.ProbeError, match="HipError"):
        w.ask("bus_id", 10 ** 6)
    assert w._child is None
    assert w.ask("matrix_bytes") > 0
    w.close()


def test_the_matrix_rate_is_published():
    from yoda_scheduler_amd.models.scv import Scv
    be = FakeBackend(2, node="n")
    prober = FailingProber(be, matrix={1: (0, 40.25)})
    agent = SnifferAgent(None, "n", be, probe=True, prober=prober, probe_matrix=True)
    assert "matrixTflops" not in agent.build().to_json()["status"]["amd"]["cards"][0]        # not measured
    agent.run_probes()
    obj = agent.build().to_json()
    assert [c["matrixTflops"] for c in obj["status"]["amd"]["cards"]] == [2500.0, 40.2]
    assert [c.matrix_tflops for c in Scv.from_json(obj).status.card_list] == [2500.0, 40.2]


def test_a_probing_process_that_cannot_be_killed_is_left(monkeypatch):
    """One that hangs in the driver outlives a kill and holds its pipes: the agent goes on."""
    from yoda_scheduler_amd.sniffer import probe

    class Hung:
        returncode = None

        def __init__(self, *args, **kw):
            out, self.held = os.pipe()
            into, give = os.pipe()
            self.stdout, self.stdin, self.read = os.fdopen(out), os.fdopen(give, "w"), into
            self.kills = 0

        def kill(self):
            self.kills += 1

        def wait(self, timeout):
            raise subprocess.TimeoutExpired("hung", timeout)

    monkeypatch.setattr(probe.subprocess, "Popen", Hung)
    w = probe.Worker(timeout=0.2)
    with pytest.raises(probe.ProbeError, match="no answer in 0.2 s"):
        w.ask("matrix", 0)
    assert w._child is None


@pytest.mark.parametrize("said", ["", "{\\\"value", "{}"])
def test_an_answer_that_is_cut_off_is_none(monkeypatch, said):
    from yoda_scheduler_amd.sniffer import probe
    real = subprocess.Popen
    monkeypatch.setattr(probe.subprocess, "Popen", lambda cmd, **kw: real(["sh", "-c", f'read q; printf "{said}"'], **kw))
    w = probe.Worker(timeout=60)
    with pytest.raises(probe.ProbeError, match="the probing process ended .status 0"):
        w.ask("matrix", 0)


def test_an_answer_reaches_a_process_with_many_open_files():
    """More than select() counts to."""
    import resource
    from yoda_scheduler_amd.sniffer import probe
    soft, hard = resource.getrlimit(resource.RLIMIT_NOFILE)
    if hard != resource.RLIM_INFINITY and hard < 2048:
        pytest.skip("few files allowed")
    resource.setrlimit(resource.RLIMIT_NOFILE, (2048, hard))
    held = []
    try:
        held = [os.open("/dev/null", os.O_RDONLY) for _ in range(1100)]
        w = probe.Worker(timeout=60)
        assert w.ask("matrix_bytes") > 0
        w.close()
    finally:
        for fd in held:
            os.close(fd)
        resource.setrlimit(resource.RLIMIT_NOFILE, (soft, hard))


def test_an_error_that_says_nothing_about_the_card_counts_for_nothing():
    """No memory (a tenant was quicker) and a fault of the program leave a card's failures as they are."""
    from yoda_scheduler_amd.ops.hip import HipError
    from yoda_scheduler_amd.sniffer import probe
    be = FakeBackend(4, node="n")
    prober = FailingProber(be, matrix={0: probe.ProbeError("AttributeError: no operators", of_card=False),
                                       1: probe.ProbeError("the probing process ended")},
                           pattern={2: probe.ProbeError("hipError 2", of_card=False)})
    agent = SnifferAgent(None, "n", be, probe=True, prober=prober, fail_threshold=2, probe_matrix=True)
    agent.run_probes()
    res = agent.run_probes()
    assert all("error" in res[i] for i in (0, 1, 2))
    assert [res[i]["fail_streak"] for i in range(4)] == [0, 2, 0, 0]
    prober.fails = {"matrix": {1: probe.ProbeError("hipError 2", of_card=False)}}
    assert agent.run_probes()[1]["fail_streak"] == 2                   # neither cleared nor counted
    assert HipError("x").code == 0
    w = probe.Worker(timeout=60)
    for what, args, of_card in (("nothing of the kind", (), False), ("bus_id", (10 ** 6,), True)):
        with pytest.raises(probe.ProbeError) as e:
            w.ask(what, *args)
        assert e.value.of_card is of_card
    w.close()


def test_a_rate_is_not_published_after_the_check_failed():
    be = FakeBackend(1, node="n")
    prober = FailingProber(be)
    agent = SnifferAgent(None, "n", be, probe=True, prober=prober, probe_matrix=True)
    agent.run_probes()
    assert agent.build().status.card_list[0].matrix_tflops == 2500.0
    prober.fails["matrix"] = {0: RuntimeError("hipError 700")}
    agent.run_probes()
    assert agent.build().status.card_list[0].matrix_tflops == 0.0
