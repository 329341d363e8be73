"""The distillation example on the host and on the GPU."""

from __future__ import annotations

import pytest

import _example_checks


def test_learns_on_the_host(cpu):
    _example_checks.learns("cpu")


def test_serves_on_the_host(cpu):
    _example_checks.serves("cpu")


def test_command(cpu, capsys):
    _example_checks.load().main(["--batch", "1", "--tokens", "24", "--steps", "2", "--vocab", "60",
                                 "--kept", "4", "--window", "5", "--sinks", "1", "--generate", "3"])
    assert "in 2 steps" in capsys.readouterr().out


@pytest.mark.gpu
def test_learns(gpu):
    _example_checks.learns("cuda")


@pytest.mark.gpu
def test_serves(gpu):
    _example_checks.serves("cuda")
