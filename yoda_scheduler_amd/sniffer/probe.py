"""The GPU probes of :mod:`..ops.hip` in a process of their own.

A process that has run a kernel keeps a context on every card: HBM that no tenant gets, and an entry in the driver's
process list. An agent that probed by itself would find each card busy with its own process from then on and probe
none a second time. So :class:`Worker` starts ``python -m yoda_scheduler_amd.sniffer.probe``, which answers one
question a line (JSON both ways) and ends with its input, and a card that hangs or takes its process down costs one answer.
"""
from __future__ import annotations

import json
import os
import select
import subprocess
import sys
from pathlib import Path
from typing import Any, Optional

from ..ops import hip

QUESTIONS = {
    "count": lambda: hip.device_count(),
    "bus_id": lambda d: hip.pci_bus_id(d),
    "bandwidth_gbps": lambda d, nbytes: float(hip.hbm_bandwidth(d, nbytes, 5)["read_gbps"]),
    "pattern_errors": lambda d, nbytes: int(hip.hbm_pattern_check(d, nbytes)["errors"]),
    "matrix_bytes": lambda: hip.matrix_check_bytes(),
    "matrix": lambda d: [(r := hip.matrix_check(d))["errors"], r["tflops"]],
}


_OUT_OF_MEMORY = 2                    # hipErrorOutOfMemory: a tenant was quicker


class ProbeError(RuntimeError):
    """A probe that could not be run to its end; ``of_card``: for all that is known, because of the card."""

    def __init__(self, message: str, of_card: bool = True) -> None:
        super().__init__(message)
        self.of_card = of_card


class Worker:
    """The process that probes: started by the first question, ended by :meth:`close` or with this one."""

    def __init__(self, timeout: float = 120.0) -> None:
        self.timeout = timeout
        self._child: Optional[subprocess.Popen] = None

    def ask(self, what: str, *args: Any) -> Any:
        if self._child is None:
            root = str(Path(__file__).resolve().parents[2])
            env = dict(os.environ, PYTHONPATH=os.pathsep.join(p for p in (root, os.environ.get("PYTHONPATH")) if p))
            self._child = subprocess.Popen([sys.executable, "-m", __name__], stdin=subprocess.PIPE,
                                           stdout=subprocess.PIPE, text=True, env=env)
        child = self._child
        line, why = "", "the probing process ended"
        try:
            child.stdin.write(json.dumps([what, *args]) + "\n")
            child.stdin.flush()
            # (an answer is one write of one line)
            ready = select.poll()
            ready.register(child.stdout, select.POLLIN)
            if ready.poll(self.timeout * 1000):
                line = child.stdout.readline()
            else:
                why = f"no answer in {self.timeout:g} s, the probing process was killed"
                child.kill()
        except OSError:
            pass
        if not line.endswith("\n"):                    # nothing, or cut off
            self.close()
            raise ProbeError(f"{what}{args}: {why} (status {child.returncode})")
        answer = json.loads(line)
        if "error" in answer:
            if answer["hip"]:                         # it may stay with the process: the next card gets a new one
                self.close()
            raise ProbeError(f"{what}{args}: {answer['error']}", of_card=answer["of_card"])
        return answer["value"]

    def close(self) -> None:
        child, self._child = self._child, None
        if child is None:
            return
        try:
            child.stdin.close()
        except OSError:
            pass
        for _ in range(2):
            try:
                child.wait(10.0)
                break
            except subprocess.TimeoutExpired:          # after a kill: it hangs in the driver, and is left to it
                child.kill()
        child.stdout.close()

    def __del__(self) -> None:
        self.close()


def main() -> int:
    # what a library prints goes to stderr, so that answers alone reach stdout
    answers = os.fdopen(os.dup(1), "w")
    os.dup2(2, 1)
    for line in sys.stdin:
        what, *args = json.loads(line)
        try:
            answer = {"value": QUESTIONS[what](*args)}
        except Exception as e:  # noqa: BLE001 - said to the one who asked
            of_hip = isinstance(e, hip.HipError)
            answer = {"error": f"{type(e).__name__}: {e}", "hip": of_hip, "of_card": of_hip and e.code != _OUT_OF_MEMORY}
        print(json.dumps(answer), file=answers, flush=True)
    return 0


if __name__ == "__main__":
    sys.exit(main())
