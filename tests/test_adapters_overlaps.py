"""netra_adapters_add refuses every overlap of what it writes with what it reads but out in y's place (before any launch)."""
import pytest

from netra_moe import layers, paths
from test_layers_host import A, B, D, refused

pytestmark = pytest.mark.skipif(not paths.layers_library().is_file(), reason="library not built")
T, L, R, N, K = 40, 3, 100, 128, 8192
X, Y, OUT, WS, PA, PB, SCALE, PLAN = A, 6 * A, 7 * A, 8 * A, B, D, 4 * A, 5 * A


def sizes():
    lib = layers.library()
    return {"x": 2 * T * K, "y": 2 * T * N, "out": 2 * T * N, "ws": lib.netra_adapters_add_workspace(T, L, R, N, K),
            "pa": lib.netra_adapters_packed_bytes(L, R, N, K, 0), "pb": lib.netra_adapters_packed_bytes(L, R, N, K, 1),
            "scale": 4 * L, "plan": lib.netra_adapters_plan_bytes(T, L)}


@pytest.mark.parametrize("written,other", [(w, o) for w in ("out", "ws") for o in ("x", "y", "out", "ws", "pa", "pb", "scale", "plan")
                                           if w != o and (w, o) != ("out", "y")])  # (out and y: test_adapters_host.py)
@pytest.mark.parametrize("end", ["first", "last"])
def test_refusals(written, other, end):
    """The written range begins with the other one's last 16 bytes, or ends with its first."""
    at = dict(x=X, y=Y, out=OUT, ws=WS, pa=PA, pb=PB, scale=SCALE, plan=PLAN)
    n = sizes()
    at[written] = at[other] + n[other] // 16 * 16 - 16 if end == "last" and n[other] >= 16 else at[other] - n[written] // 16 * 16 + 16
    text = refused("netra_adapters_add", at["x"], 0, K, at["pa"], at["pb"], at["scale"], at["plan"], at["y"], N, at["out"], N, T, L, R, N, K,
                   at["ws"], n["ws"], None)
    assert "shares memory" in text


def test_the_workspace_is_as_long_as_the_call_needs():
    """Of a longer one the end may be anything; a call that needs none has none that could overlap."""
    lib = layers.library()
    need = sizes()["ws"]
    args = (X, 0, K, PA, PB, SCALE, PLAN, Y, N)
    assert "shares memory" in refused("netra_adapters_add", *args, WS + need - 16, N, T, L, R, N, K, WS, need + 4096, None)
    assert lib.netra_adapters_add_workspace(T, L, 16, N, 128) == 0
