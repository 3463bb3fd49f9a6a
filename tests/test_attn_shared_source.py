"""What the softmax warps of the attention over shared pages hand to the tensor cores: all lanes' stores come before the arrival of one of them."""
import os
import re

SOURCE = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "rexl3_b200", "ops", "csrc", "attention_shared.cu")


def test_a_warp_meets_between_its_stores_and_the_arrival():
    text = open(SOURCE).read()
    arrivals = [m.start() for m in re.finditer(r"mbar_arrive\(&p_ready\[", text)]
    assert len(arrivals) == 2                                # warps with pairs, and without
    for at in arrivals:
        stores = text.rindex("tail(j)", 0, at)               # the zeros over keys that nobody sees
        assert "__syncwarp();" in text[stores:at]
