"""Trains a gated recurrent language model with 8-bit AdamW, then continues prompts with its weights in 8 bits.

The session trains through the captured step; ``answerer`` then reads a prompt in one scan and goes on a token at a time from the states.
"""
import argparse
import os
import sys
import time

import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))
from autodist_b200 import AutoDist, strategy as S  # noqa: E402
from autodist_b200.models.recurrent_lm import RecurrentLM, RecurrentLMConfig, cyclic_tokens  # noqa: E402
from autodist_b200.optim import ListAdamW  # noqa: E402
from autodist_b200.resource_spec import ResourceSpec  # noqa: E402


def main():
    ap = argparse.ArgumentParser()
    ap.add_argument("--gpus", type=int, default=int(os.environ.get("WORLD_SIZE", "1")))
    ap.add_argument("--batch_size", type=int, default=16, help="per GPU")
    ap.add_argument("--seq_len", type=int, default=64)
    ap.add_argument("--steps", type=int, default=60)
    ap.add_argument("--lr", type=float, default=None, help="2e-3 for the tiny model, 2e-4 for the full one")
    ap.add_argument("--tokens", type=int, default=20, help="to continue the prompt by")
    ap.add_argument("--state_bits", type=int, default=8, choices=(8, 32))
    ap.add_argument("--tiny", action="store_true")
    args = ap.parse_args()
    n = args.gpus
    cfg = RecurrentLMConfig.tiny() if args.tiny else RecurrentLMConfig()
    ad = AutoDist(resource_spec=ResourceSpec.local(num_gpus=n if torch.cuda.is_available() else 0, num_cpus=n), strategy_builder=S.AllReduce())
    data = cyclic_tokens(args.batch_size * n, args.seq_len, cfg.vocab_size)
    with ad.scope():
        torch.manual_seed(0)
        model = RecurrentLM(cfg)
        feeds = {k: ad.placeholder((None, args.seq_len), torch.int64, name=k) for k in ("x", "y")}
        loss = model(**feeds)
        train_op = ListAdamW(model.parameters(), lr=args.lr or (2e-3 if args.tiny else 2e-4), state_bits=args.state_bits).minimize(loss)
        sess = ad.create_distributed_session()
        t0 = time.time()
        for step in range(1, args.steps + 1):
            value, _ = sess.run([loss, train_op], {feeds[k]: data[k] for k in feeds})
            if sess.rank == 0 and step % 10 == 0:
                print(f"step {step} loss {float(value):.3f} {10 * data['x'].numel() / (time.time() - t0):.0f} tokens/s", flush=True)
                t0 = time.time()
        if sess.rank == 0:
            prompt = data["x"][:2, :16].to(next(model.parameters()).device)
            answer = model.answerer()
            logits, states = answer(prompt)
            said = []
            for _ in range(args.tokens):
                token = logits.argmax(-1, keepdim=True)
                said.append(token)
                logits, states = answer(token, states)
            said = torch.cat(said, 1).cpu()
            want = torch.stack([data["x"][i, 16:16 + args.tokens] for i in range(2)])
            print(f"continued {said.shape[1]} tokens, {float((said == want[:, :said.shape[1]]).float().mean()):.2f} of them as the sequence goes on")
        sess.close()


if __name__ == "__main__":
    main()
