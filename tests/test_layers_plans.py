"""CPU-only: the sizes of tests/plan_cases.py, which the GPU tests run, take the kernels that they are there for, and all kernels
of the plans are among them (tests/cpp/plans_check.cpp)."""
import os
import random
import subprocess

import pytest

from plan_cases import MX4, PAIRS


@pytest.fixture(scope="module")
def plans():
    at = os.path.join(os.path.dirname(os.path.abspath(__file__)), "cpp")
    subprocess.check_call(["make", "-C", at, "-B", "plans_check"], stdout=subprocess.DEVNULL, stderr=subprocess.DEVNULL)

    def ask(lines):
        out = subprocess.run([os.path.join(at, "plans_check")], input="\n".join(lines) + "\n", capture_output=True, text=True)
        assert out.returncode == 0
        return [line.strip() for line in out.stdout.strip().split("\n")]
    return ask


def sizes(rng, *most):
    return tuple(int(round(m ** rng.random())) for m in most)


def kinds_of_mx4(plan):
    name, a, b = plan.split()[:3]
    return (name, a, b != "1") if name == "tiles" else (name, a, b)


def test_sizes_of_4_bit_products_take_every_kernel(plans):
    assert plans(["mx4 %d %d %d %d" % (*shape, not codes) for shape, codes, _ in MX4]) == [plan for _, _, plan in MX4]
    rng = random.Random(1)
    lines = ["mx4 %d %d %d %d" % (*sizes(rng, 20000, 20000, 40000), rng.random() < 0.5) for _ in range(20000)]
    assert {kinds_of_mx4(p) for p in plans(lines)} == {kinds_of_mx4(p) for _, _, p in MX4}


def kinds_of_pairs(plan):
    w = plan.split()
    return set() if w[0] == "whole" else {(i, w[4 * i], w[4 * i + 2] != "1") for i in range(3)}


def test_sizes_of_orthogonalised_updates_take_every_kernel(plans):
    assert plans(["orth %d %d %d" % shape for shape, _ in PAIRS]) == [plan for _, plan in PAIRS]
    rng = random.Random(2)
    lines = ["orth %d %d %d" % ((rng.choice([1, 1, *sizes(rng, 64)]),) + sizes(rng, 9000, 9000)) for _ in range(20000)]
    assert set().union(*map(kinds_of_pairs, plans(lines))) == set().union(*(kinds_of_pairs(p) for _, p in PAIRS))
