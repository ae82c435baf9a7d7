"""Log probabilities straight from a head: the refusals that need no GPU."""
import ctypes

from purebee_amd import native


def test_null_arguments_are_refused():
    L = native.load_library()
    size = ctypes.c_size_t()
    for rc in (L.pbx_linear_logprobs_workspace(None, None, 1, 0, ctypes.byref(size)),
               L.pbx_linear_logprobs_dev(None, None, None, 1, None, None, None, None, None, 0),
               L.pbx_linear_logprobs_grad_dev(None, None, None, 1, None, None, None, None, None, 0)):
        assert rc == -1
        assert b"ctx is NULL" in L.pbx_last_error(None)
