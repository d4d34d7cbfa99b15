"""Linear attention and block_norm on the CPU: what the PyTorch operators, the Python functions and the C ABI do with a call
before anything runs on a device."""
import sffft_b200 as sf


def test_the_wait_limit_refuses_what_it_does_not_know():
    f = sf.lib().sffft_debug_linear_attention
    for bad in ((-1, 0), (1000001, 0), (2000, -1), (2000, 4), (0, 1)):
        assert f(*bad) == sf.ERR_INVALID_ARGUMENT
    assert f(2000, 3) == sf.OK and f(0, 0) == sf.OK
