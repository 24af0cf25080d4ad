"""The recurrent language model on a GPU: the kernels together, against the same model's expressions on the host."""
import copy

import pytest
import torch

pytestmark = pytest.mark.gpu


def test_losses_and_gradients_are_the_hosts():
    """bf16 activations against fp32 ones: a loss and gradients a few hundredths apart."""
    from autodist_b200.models.recurrent_lm import RecurrentLM, RecurrentLMConfig, cyclic_tokens
    cfg = RecurrentLMConfig(vocab_size=64, width=64, units=96, layers=3)
    torch.manual_seed(1)
    host = RecurrentLM(cfg)
    there = copy.deepcopy(host).cuda()
    data = cyclic_tokens(5, 70, cfg.vocab_size)
    a, b = host(data["x"], data["y"]), there(data["x"].cuda(), data["y"].cuda())
    assert abs(float(a) - float(b)) < 0.02 * float(a)
    a.backward()
    b.backward()
    for (name, p), q in zip(host.named_parameters(), there.parameters()):
        assert float((p.grad - q.grad.cpu()).norm()) < 0.05 * float(p.grad.norm()) + 1e-4, name


@pytest.mark.parametrize("bits", [8, 32])
def test_trains_through_a_session_and_answers_in_eight_bits(bits):
    from autodist_b200 import AutoDist, strategy as S
    from autodist_b200.autodist import _reset_default_autodist
    from autodist_b200.models.recurrent_lm import RecurrentLM, RecurrentLMConfig, cyclic_tokens
    from autodist_b200.ops import functional as F
    from autodist_b200.optim import ListAdamW
    from autodist_b200.resource_spec import ResourceSpec
    _reset_default_autodist()
    ad = AutoDist(resource_spec=ResourceSpec.local(num_gpus=1), strategy_builder=S.AllReduce())
    cfg = RecurrentLMConfig.tiny()
    data = cyclic_tokens(16, 64, cfg.vocab_size)
    with ad.scope():
        torch.manual_seed(0)
        model = RecurrentLM(cfg)
        feeds = {k: ad.placeholder((None, 64), torch.int64, name=k) for k in data}
        loss = model(**feeds)
        train_op = ListAdamW(model.parameters(), lr=2e-3, state_bits=bits).minimize(loss)
        sess = ad.create_distributed_session()
        losses = [float(sess.run([loss, train_op], {feeds[k]: data[k] for k in feeds})[0]) for _ in range(60)]
        answer = model.answerer()
        ids = data["x"].cuda()
        logits, states = answer(ids[:, :16])
        right = 0
        for t in range(16, 48):
            right += int((logits.argmax(-1) == ids[:, t]).sum())
            logits, states = answer(ids[:, t:t + 1], states)
        sess.close()
    _reset_default_autodist()
    F.check_errors()
    assert losses[-1] < 0.2 * losses[0] and right >= 0.95 * 32 * 16
