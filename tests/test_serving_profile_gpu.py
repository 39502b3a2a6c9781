"""The serving operators under the engine's profiler: launchers alone are timed, each in its class."""
import pytest
import torch

import test_adapters_gpu as adapters
import test_shared_attention_gpu as attention

pytestmark = pytest.mark.gpu


def test_what_the_profiler_reports():
    from logssms_b200.ops.profiler import PROFILER
    from logssms_b200.sampling import edit_logits
    s = attention.make([(300, [1, 5, 64])], 8, 2, 64, 64, torch.bfloat16)
    a = adapters.make(400, 65, 64, 3, 13, torch.bfloat16, [t % 3 for t in range(400)])
    plain = attention.call(s), attention.K().add_adapters(a["y"], a["x"], a["a"], a["b"], a["index"], a["scales"])
    logits = torch.zeros((2, 50), device="cuda")
    PROFILER.reset()
    PROFILER.enable()
    try:
        timed = attention.call(s), attention.K().add_adapters(a["y"], a["x"], a["a"], a["b"], a["index"], a["scales"])
        edit_logits(logits)
        report = PROFILER.report()
    finally:
        PROFILER.disable()
        PROFILER.reset()
    assert all(torch.equal(x, y) for x, y in zip(plain, timed))
    assert {name: entry["launches"] for name, entry in report["kernels"].items()} == {
        "attention_shared.lb_attention_shared": 1, "adapters.lb_add_adapters": 1, "logit_rules.lb_logit_rules": 1}
    assert set(report["classes"]) == {"attention", "products", "sampling"}
