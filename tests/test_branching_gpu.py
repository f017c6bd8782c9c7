"""Forks, shrinks and shared steps of engines on the GPU: the tests that any device runs, run there."""

import pytest

import test_branching
import test_branching_requests

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("length", [1, 30, 64, 65])
def test_choices_fork(length):
    test_branching.test_choices_fork(length)


@pytest.mark.parametrize("hipgraph", [False, True])
def test_shared_prefix_steps(hipgraph, monkeypatch):
    test_branching.test_shared_prefix_steps(hipgraph, monkeypatch)


def test_shrinks_between_steps(monkeypatch):
    test_branching.test_shrinks_between_steps(monkeypatch)


@pytest.mark.parametrize("name", [
    "test_a_fork_of_something_else_is_prefilled", "test_a_fork_of_an_ended_request", "test_forks_that_wait_for_nobody",
    "test_forks_of_a_fork", "test_forks_under_cache_pressure", "test_the_loop_forks_choices"])
def test_forks(name):
    getattr(test_branching, name)()


@pytest.mark.parametrize("fork", [False, True])
def test_an_empty_prompt_is_refused_by_itself(fork):
    test_branching_requests.test_an_empty_prompt_is_refused_by_itself(fork)
