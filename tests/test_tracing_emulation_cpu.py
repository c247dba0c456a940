"""Tracing, torch.compile and torch.func on the norms and the router's balance loss, with the library's host side and kernels
emulated on the host (bodies in tests/tracing_cases.py)."""

import pytest

import tracing_cases as cases
import train_ops_emu


@pytest.fixture(autouse=True)
def _emulation():
    with train_ops_emu.installed():
        yield


@pytest.mark.parametrize("mode", ["real", "fake", "symbolic"])
@pytest.mark.parametrize("name", ["layer", "rms", "balance"])
def test_make_fx(name, mode):
    cases.case_make_fx("cpu", name, mode)


def test_make_fx_of_a_bare_norm():
    cases.case_make_fx_of_a_bare_norm("cpu")


@pytest.mark.parametrize("name", ["layer", "rms", "balance"])
def test_compile(name):
    cases.case_compile("cpu", name)


def test_compile_modules():
    cases.case_compile_modules("cpu")


def test_meta():
    cases.case_meta("cpu")


@pytest.mark.parametrize("name", ["layer", "rms", "balance"])
def test_functional_gradients(name):
    cases.case_functional_gradients("cpu", name)


def test_second_derivative_is_refused():
    cases.case_second_derivative_is_refused("cpu")


def test_outputs_are_as_described():
    cases.case_outputs_are_as_described("cpu")


def test_plain_calls_take_the_short_way():
    cases.case_plain_calls_take_the_short_way("cpu")


def test_lazy_negatives():
    cases.case_lazy_negatives("cpu")


def test_forward_over_reverse():
    cases.case_forward_over_reverse("cpu")


def test_operators_check_what_belongs_together():
    cases.case_operators_check_what_belongs_together("cpu")
