"""What needs no GPU of the sequence operators' unusual cases."""


def test_waits_are_made_to_run_out_only_on_request():
    from dwconv_b200 import _lib
    expire = _lib.lib.dwconv_b200_debug_expire
    assert expire(1) == 0 and expire(2) == 1 and expire(5) == 2 and expire(0) == 0
