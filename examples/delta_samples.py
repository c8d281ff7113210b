"""Several answers to one prompt from a hybrid of gated delta rule and attention.

    python examples/delta_samples.py [--layers 8] [--width 512] [--prompt-len 300] [--samples 4] [--max-tokens 24]

Defines a small architecture through the package's registry - layers whose mixer is the gated delta rule, every
fourth one grouped-query attention - writes a model folder with random weights, runs a prompt once and continues it several times:
the pages of the attention layers are shared, a begun page and the delta rule's states are copied.  Then the pages in
use are brought to the front of their pool.  Needs a B200."""

from __future__ import annotations

import argparse
import sys
import tempfile
from dataclasses import asdict, dataclass, fields
from pathlib import Path

sys.path.insert(0, str(Path(__file__).resolve().parent.parent))

NAME = "DeltaHybridForCausalLM"


@dataclass(frozen=True)
class DeltaHybridConfig:
    width: int
    layers: int
    vocab: int
    heads: int              # of values; the attention layers' query heads
    qk_heads: int           # of the delta rule's keys and queries; the attention layers' kv heads
    dim: int
    vdim: int
    taps: int = 4
    attention_every: int = 4
    eps: float = 1e-6
    theta: float = 10000.0

    @classmethod
    def from_dict(cls, d):
        return cls(**{f.name: d[f.name] for f in fields(cls) if f.name in d})

    def to_dict(self):
        return {"architectures": [NAME], **asdict(self)}

    def attends(self, layer: int) -> bool:
        return layer % self.attention_every == self.attention_every - 1

    def build_spec(self):
        from from_scratch_inference_engine_b200.config import LayerCall, LayerSpec, ModelSpec, PartSpec
        norm = PartSpec("rmsnorm", {"width": self.width, "eps": self.eps})
        delta = PartSpec("gated_delta_rule", {
            "hidden_size": self.width, "heads": self.heads, "qk_heads": self.qk_heads, "dim": self.dim, "vdim": self.vdim,
            "taps": self.taps, "eps": self.eps})
        attention = PartSpec("gqa_attention", {
            "hidden_size": self.width, "num_heads": self.heads, "num_kv_heads": self.qk_heads, "head_dim": self.dim,
            "qkv_bias": False, "window": 0,
            "position": PartSpec("rotary", {"theta": self.theta, "rotary_dim": self.dim, "max_position": 0})})
        layers = tuple(LayerSpec(
            prefix=f"layers.{i}.", arrangement="prenorm", mixer=attention if self.attends(i) else delta,
            feed_forward=PartSpec("swiglu", {"hidden_size": self.width, "intermediate_size": 2 * self.width}),
            mixer_norm=norm, feed_forward_norm=norm) for i in range(self.layers))
        return ModelSpec(NAME, self.width, self.vocab, 0, "embed.weight", None, norm, "final_norm.", layers,
                         tuple(LayerCall(i) for i in range(self.layers)))


def main(argv=None) -> int:
    parser = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    parser.add_argument("--layers", type=int, default=8)
    parser.add_argument("--width", type=int, default=512)
    parser.add_argument("--prompt-len", type=int, default=300)
    parser.add_argument("--samples", type=int, default=4)
    parser.add_argument("--max-tokens", type=int, default=24)
    parser.add_argument("--temperature", type=float, default=0.9)
    parser.add_argument("--seed", type=int, default=0)
    args = parser.parse_args(argv)

    import random
    from from_scratch_inference_engine_b200 import LLM, GenerationConfig, register_architecture, write_random_model
    register_architecture(NAME, DeltaHybridConfig)
    config = DeltaHybridConfig(width=args.width, layers=args.layers, vocab=2048, heads=args.width // 64,
                               qk_heads=max(1, args.width // 128), dim=64, vdim=64)
    rng = random.Random(args.seed)
    prompt = [rng.randrange(config.vocab) for _ in range(args.prompt_len)]
    with tempfile.TemporaryDirectory() as folder:
        llm = LLM(write_random_model(Path(folder) / "model", config, seed=1, std=0.05), block_size=16, num_blocks=1024,
                  max_batch=max(8, args.samples), eos_id=-1)
        answers = llm.generate_samples(prompt, args.samples, GenerationConfig(
            max_tokens=args.max_tokens, temperature=args.temperature, seed=args.seed))
        stats = llm.engine.stats()
    for index, answer in enumerate(answers):
        print(f"[{index}] {','.join(map(str, answer))}")
    print(f"prompt tokens run: {stats['tokens_prefilled']} for {args.samples} answers to a prompt of {len(prompt)}")
    print(f"pages in use after compaction: {llm.engine.compact()}")
    return 0


if __name__ == "__main__":
    sys.exit(main())
