"""CPU checks of the block operators' entry points."""


def test_plan_set_status_refuses_a_null_plan(nkv):
    assert nkv.lib().nkv_attend_plan_set_status(None, 0) == 6
