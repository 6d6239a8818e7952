// GPU check of the text encoder over a cache of two sequences: calls of unequal pieces in flight at once against the same
// calls one after the other, and a recorded step that only one sequence takes part in against an eager call. Prints one
// JSON object with the largest differences.
//   node extend_overlap.mjs WEIGHTS.safetensors CACHE_BITS
import path from "path";
import { fileURLToPath, pathToFileURL } from "url";

const here = path.dirname(fileURLToPath(import.meta.url));
const js = path.resolve(here, "..", "..", "nanosaur2-web_amd", "js");
const mod = (f) => import(pathToFileURL(path.join(js, f)).href);

async function main() {
  const { GPU } = await mod("device.js");
  const { SafeTensors } = await mod("weights.js");
  const { Gemma3 } = await mod("gemma3.js");
  const ops = await mod("ops.js");
  const [file, bits] = [process.argv[2], Number(process.argv[3])];
  const gpu = await GPU.create({});
  const st = await SafeTensors.open(file);
  const te = await Gemma3.load(gpu, st);
  const pieces = [[[1, 2, 3, 4, 5], [6, 7]], [[], [8, 9, 10]], [[11], [12]]];
  // every row that belongs to a token
  const hidden = async (h, piece) => {
    const all = await gpu.read(h);
    h.release();
    const L = Math.max(...piece.map((t) => t.length));
    return piece.flatMap((t, b) => t.map((_, i) => Array.from(all.subarray((b * L + i) * 640, (b * L + i + 1) * 640))));
  };
  const together = te.newCache({ batch: 2, capacity: 40, bits, sinks: 1 });
  const apart = te.newCache({ batch: 2, capacity: 40, bits, sinks: 1 });
  const hs = await Promise.all(pieces.map((p) => te.extend(together, p)));
  let overlap = 0;
  const worst = (a, b) => a.reduce((m, row, i) => row.reduce((n, x, j) => Math.max(n, Math.abs(x - b[i][j]) || (x === b[i][j] ? 0 : Infinity)), m), 0);
  for (let i = 0; i < pieces.length; i++) {
    overlap = Math.max(overlap, worst(await hidden(hs[i], pieces[i]), await hidden(await te.extend(apart, pieces[i]), pieces[i])));
  }
  const lengths = [[...together.lengths], [...apart.lengths]];
  const step = te.captureStep(together);
  let recorded = 0;
  for (const [id, active] of [[13, [true, true]], [14, [false, true]], [15, [true, false]], [16, [true, true]]]) {
    const emb = te.embed(await st.rows("model.embed_tokens.weight", [id, id + 1]), 2);
    ops.elementwise(gpu, "copy", emb, null, step.input);
    emb.release();
    step.launch(active);
    const all = await gpu.read(step.output);
    const rows = [0, 1].filter((b) => active[b]).map((b) => Array.from(all.subarray(b * 640, (b + 1) * 640)));
    const piece = [0, 1].map((b) => (active[b] ? [id + b] : []));
    recorded = Math.max(recorded, worst(rows, await hidden(await te.extend(apart, piece), piece)));
  }
  lengths.push([...together.lengths], [...apart.lengths]);
  step.destroy();
  together.destroy();
  apart.destroy();
  te.unload();
  if (st.close) st.close();
  process.stdout.write(JSON.stringify({ overlap, recorded, lengths }) + "\n");
}

main().catch((e) => {
  process.stderr.write(String(e && e.stack ? e.stack : e) + "\n");
  process.exit(1);
});
