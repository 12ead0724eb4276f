"""CPU: host-side queries of the packed-prompt and shared-prefix attention"""


def test_prefix_form_refuses_what_the_call_refuses(built_lib):
    f = built_lib.ifh_attn_prefix_form
    for bad in ((0, 1, 10, 4, 1, 10), (1, 0, 10, 4, 1, 10), (1, 1, 0, 4, 1, 10), (1, 1, 10, 4, 3, 10), (1, 1, 10, 4, 0, 10), (1, 1, 10, 4, 1, 0),
                (1 << 24, 1, 10, 4, 1, 10)):
        assert f(*bad) == -1, bad
    assert f(2, 1, 333, 4, 1, 64) >= 0
