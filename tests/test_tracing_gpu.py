"""Tracing, torch.compile and torch.func on the norms and the router's balance loss on a B200 (bodies in tests/tracing_cases.py)."""

import pytest

import tracing_cases as cases

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("mode", ["real", "fake", "symbolic"])
@pytest.mark.parametrize("name", ["layer", "rms", "balance"])
def test_make_fx(name, mode):
    cases.case_make_fx("cuda", name, mode)


def test_make_fx_of_a_bare_norm():
    cases.case_make_fx_of_a_bare_norm("cuda")


@pytest.mark.parametrize("name", ["layer", "rms", "balance"])
def test_compile(name):
    cases.case_compile("cuda", name)


def test_compile_modules():
    cases.case_compile_modules("cuda")


def test_meta():
    cases.case_meta("cuda")


@pytest.mark.parametrize("name", ["layer", "rms", "balance"])
def test_functional_gradients(name):
    cases.case_functional_gradients("cuda", name)


def test_second_derivative_is_refused():
    cases.case_second_derivative_is_refused("cuda")


def test_outputs_are_as_described():
    cases.case_outputs_are_as_described("cuda")


def test_plain_calls_take_the_short_way():
    cases.case_plain_calls_take_the_short_way("cuda")


def test_lazy_negatives():
    cases.case_lazy_negatives("cuda")


def test_forward_over_reverse():
    cases.case_forward_over_reverse("cuda")


def test_operators_check_what_belongs_together():
    cases.case_operators_check_what_belongs_together("cuda")
