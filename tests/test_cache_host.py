"""The text encoder's calls over a key/value cache on the CPU (tests/js/cache_checks.mjs): positions of tokens when
calls overlap, fail, or meet a recorded step. What runs on the GPU from there on is held to 64 bits elsewhere."""

import json
import os
import subprocess

import pytest

CHECKS = os.path.join(os.path.dirname(os.path.abspath(__file__)), "js", "cache_checks.mjs")


@pytest.fixture(scope="module")
def checks():
    p = subprocess.run(["node", CHECKS], capture_output=True, text=True, timeout=60)
    assert p.returncode == 0, p.stderr
    return json.loads(p.stdout.strip().splitlines()[-1])


def test_calls_in_flight_take_positions_in_their_order(checks):
    """Whatever order their embedding rows arrive in, the second call's tokens come behind the first's."""
    assert checks["overlap"] == {"ends": ["ok", "ok"], "asked": [[5, 6, 7], [8, 9]], "lengths": [5],
                                 "ran": [{"pos": [0, 1, 2], "L": 3, "rows": 3}, {"pos": [3, 4], "L": 2, "rows": 2}]}
    assert checks["batch"] == {"ends": ["ok", "ok"], "lengths": [3, 3],
                               "ran": [{"pos": [0, 1, 2, 0, -1, -1], "L": 3, "rows": 6}, {"pos": [-1, -1, 1, 2], "L": 2, "rows": 4}]}


def test_a_call_without_room_is_refused_alone(checks):
    c = checks["capacity"]
    assert c["ends"][0] == "ok" and "no room for 2 more" in c["ends"][1] and c["ends"][2] == "ok"
    assert [r["pos"] for r in c["ran"]] == [[0, 1, 2], [3]] and c["lengths"] == [4]


def test_rows_that_cannot_be_read_fail_their_call_alone(checks):
    c = checks["rows"]
    assert c["ends"] == ["no such row", "ok"] and [r["pos"] for r in c["ran"]] == [[0]] and c["lengths"] == [1]
    c = checks["late"]
    assert c["ends"] == ["ok", "no such row", "ok"] and [r["pos"] for r in c["ran"]] == [[0, 1], [2]] and c["lengths"] == [3]


def test_a_recorded_step_meets_a_call_in_flight(checks):
    """A step launched while rows are on their way takes the next position, the call those behind it; a length set back
    in between holds for the call."""
    c = checks["step"]
    assert c["ends"] == ["ok"] and c["steps"] == [[2]] and [r["pos"] for r in c["ran"]] == [[3, 4]] and c["lengths"] == [5]
    c = checks["cut"]
    assert c["ends"] == ["ok"] and [r["pos"] for r in c["ran"]] == [[1]] and c["lengths"] == [2]


@pytest.mark.parametrize("kind", ["bf16", "i4"])
def test_a_failing_launch_leaves_nothing_behind(checks, kind):
    """Whichever launch of the layer stack fails: the positions, the activations and the results of the ops before it go
    back to the pool, and no token counts. The call without a failure keeps its result alone."""
    runs = checks["failures"][kind]
    assert len(runs) > 10 and runs[-1] == ["ok", 1, 2], runs
    assert all(r == ["a launch failed", 0, 0] for r in runs[:-1]), runs


def test_ids_in_typed_arrays(checks):
    assert checks["typed"] == {"ends": ["ok"] * 3, "ran": [[0, 1, 2], [3, 4], [5]], "asked": [[5, 6, 7], [8, 9], [1]]}
