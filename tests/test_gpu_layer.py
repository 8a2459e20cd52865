"""Whole layers: token mixers and the MoE block of one library, as a model's layers use them."""
import numpy as np
import pytest

torch = pytest.importorskip("torch")
import mixer_ref as R  # noqa: E402
import oracle as O  # noqa: E402
import qe_mixer  # noqa: E402
import qe_moe  # noqa: E402

pytestmark = pytest.mark.gpu
D, HQ, HKV, DIM, HK, HV, DK = qe_moe.D, 16, 2, 256, 16, 32, 128
SEED = 20251201


class Model:
    """Two layers: attention, then the delta rule, each followed by the residual and the MoE block."""

    def __init__(self, t_max):
        g = torch.Generator(device="cuda")
        g.manual_seed(1)

        def weight(rows, cols):
            return torch.randn(rows, cols, generator=g, device="cuda") * cols ** -0.5

        self.w_qkv, self.w_o = weight((HQ + 2 * HKV) * DIM, D), weight(D, HQ * DIM)
        self.w_d, self.w_do = weight(2 * HK * DK + HV * DK, D), weight(D, HV * DK)
        self.w_gb = weight(2 * HV, D)
        self.moe = qe_moe.MoE(n_layers=2, t_max=t_max)
        for layer in range(2):
            self.moe.synth_layer(layer, SEED)
        self.att = qe_mixer.Attention(HQ, HKV, DIM, 16, rotary=64, theta=1e7, sections=(11, 11, 10), interleaved=True)
        self.delta = qe_mixer.GatedDelta(HK, HV, DK, DK, t_max=t_max)
        self.kc, self.vc = (torch.full((40, HKV, 16, DIM), float("nan"), dtype=torch.bfloat16, device="cuda") for _ in range(2))
        self.pool = torch.full((4, HV, DK, DK), float("nan"), device="cuda")

    def layers(self, x, kv_len, table, cu, slots_in, slots):
        """x [T, D] through both layers.  cu None: one token per sequence.  Also what each mixer took and gave."""
        T = x.shape[0]
        s = torch.cuda.current_stream()
        batch = qe_mixer.Batch(kv_len, table, cu)
        norm = torch.nn.functional.rms_norm
        q, k, v = (norm(x, (D,)) @ self.w_qkv.T).view(T, -1, DIM).split((HQ, HKV, HKV), 1)
        q, k = norm(q, (DIM,)), norm(k, (DIM,))
        r, a = (torch.empty(T, HQ, DIM, dtype=torch.bfloat16, device="cuda") for _ in range(2))
        self.att.append(batch, q, k, v, self.kc, self.vc, r, stream=s)
        (self.att.decode if cu is None else self.att.prompt)(batch, r, self.kc, self.vc, a, stream=s)
        x2 = x + a.view(T, -1).float() @ self.w_o.T
        y = torch.empty_like(x)
        self.moe.forward(0, x2, y, T, stream=s)
        n = norm(y, (D,))
        q, k, v = torch.nn.functional.silu(n @ self.w_d.T).split((HK * DK, HK * DK, HV * DK), 1)
        g, beta = (n @ self.w_gb.T).view(T, 2, HV).unbind(1)
        g, beta = -torch.nn.functional.softplus(g), torch.sigmoid(beta)
        d = torch.empty(T, HV, DK, device="cuda")
        args = (q, k, v, g, beta.contiguous(), self.pool, slots_in, slots)
        if cu is None:
            self.delta.decode(*args, d, stream=s)
        else:
            self.delta.prompt(*args, cu, d, stream=s)
        z2 = y + d.view(T, -1) @ self.w_do.T
        z = torch.empty_like(x)
        self.moe.forward(1, z2, z, T, stream=s)
        return z, dict(r=r, a=a, x2=x2, y=y, q=q, k=k, v=v, g=g, beta=beta, d=d)


def test_two_layers_prompt_then_tokens():
    m = Model(t_max=64)
    g = torch.Generator(device="cuda")
    g.manual_seed(2)
    table = torch.randperm(40, generator=g, device="cuda").to(torch.int32).view(2, 20)
    lens, slots = [37, 11], torch.tensor([2, 0], dtype=torch.int32, device="cuda")
    xs = [torch.randn(n + 3, D, generator=g, device="cuda") for n in lens]

    def ints(v):
        return torch.tensor(v, dtype=torch.int32, device="cuda")

    took = [[], []]  # per sequence, each call's record
    z, t = m.layers(torch.cat([x[:n] for x, n in zip(xs, lens)]), ints(lens), table, ints([0, 37, 48]), ints([-1, -1]), slots)
    took[0].append({k: v[:37] for k, v in t.items()}), took[1].append({k: v[37:] for k, v in t.items()})
    for step in range(3):
        z, t = m.layers(torch.stack([x[n + step] for x, n in zip(xs, lens)]), ints([n + step + 1 for n in lens]), table, None, slots, slots)
        for i in range(2):
            took[i].append({k: v[i: i + 1] for k, v in t.items()})
    m.att.check(), m.delta.check(), m.moe.check()
    assert bool(torch.isfinite(z).all())
    layer = O.SynthLayer(SEED, 0)
    for i in range(2):
        all_ = {k: torch.cat([x[k] for x in took[i]]) for k in took[i][0]}
        n = lens[i] + 3
        # attention of every token against the definition over the whole sequence's cache
        want, off = R.attend_batch(all_["r"], m.kc, m.vc, table[i: i + 1], [n], [0, n], DIM ** -0.5, 16)
        assert bool(((all_["a"].double() - want).abs() <= off).all())
        # the delta rule, prompt and tokens, against one recurrence from nothing
        o, S = R.delta(all_["q"].reshape(n, HK, DK), all_["k"].reshape(n, HK, DK), all_["v"].reshape(n, HV, DK), all_["g"], all_["beta"],
                       torch.zeros(HV, DK, DK, device="cuda"), True, DK ** -0.5)
        assert R.rel(all_["d"], o) <= 1e-5 and R.rel(m.pool[int(slots[i])], S) <= 1e-5
    # the MoE block on what attention made, against the oracle
    x2 = took[0][-1]["x2"].cpu().numpy()
    w = O.moe_layer(layer, x2, norm=True, residual=True)["out"]
    assert np.linalg.norm(took[0][-1]["y"].cpu().numpy() - w) <= 1e-3 * np.linalg.norm(w)
