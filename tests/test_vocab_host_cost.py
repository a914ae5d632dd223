"""What the vocabulary operators cost a graph that has none: nothing is called for them."""
import sys

import torch

import fugatensor_b200 as ft


def test_building_a_primitive_enters_no_frame_for_the_operators_flag():
    x = ft.Tensor(ft.current_engine(), ft.fp32, (4, 8), data=torch.empty(0))
    callees = []

    def watch(frame, event, arg):
        if event == "call" and frame.f_back is not None and frame.f_back.f_code.co_name == "_prim":
            callees.append(frame.f_code.co_name)

    sys.setprofile(watch)
    try:
        y = x + x
    finally:
        sys.setprofile(None)
    assert sorted(callees) == ["__init__", "_infer"] and not y._ops
