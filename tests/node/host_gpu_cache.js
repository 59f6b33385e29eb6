// GPU run of CacheAppendKernel, CacheAttentionKernel and DraftVerifyKernel in
// one command buffer. Usage: node host_gpu_cache.js <case.json>; run by
// tests/test_node_cache.py, which checks what it writes.
"use strict";
const assert = require("assert");
const fs = require("fs");
const path = require("path");
const host = require(path.join(__dirname, "..", "..", "parakeet.wgsl_amd", "host"));

async function main() {
  const spec = JSON.parse(fs.readFileSync(process.argv[2], "utf8"));
  const device = host.HipGpuDevice.create();
  const arena = new host.GpuActivationArena(device, 32 * 1024 * 1024);
  let at = 0;
  const slices = {};
  function slice(name, bytes) {
    slices[name] = arena.slice(name, at, bytes);
    at += Math.ceil(bytes / 256) * 256;
    return slices[name];
  }
  for (const [name, file] of Object.entries(spec.files)) {
    const b = fs.readFileSync(file);
    arena.upload(device, slice(name, b.byteLength), new Uint8Array(b.buffer, b.byteOffset, b.byteLength));
  }
  const { rows, sequences, heads, kvHeads, headDim, active } = spec;
  for (const name of ["rotated", "attended"]) slice(name, rows * heads * headDim * 2);
  for (const name of ["accepted", "nextTokens"]) slice(name, sequences * 4);
  const cache = Object.assign({
    rowStarts: slices.rowStarts, lengths: slices.lengths, pageTable: slices.pageTable, keys: slices.keyCache,
    values: slices.valueCache,
  }, spec.cache);
  const shape = { rows, sequences, heads, kvHeads, headDim, cache };
  const append = await host.CacheAppendKernel.create(device, arena);
  const attention = await host.CacheAttentionKernel.create(device, arena);
  const verify = await host.DraftVerifyKernel.create(device, arena);
  const dispatches = [
    append.createDispatch(Object.assign({
      label: "append", queries: slices.queries, queryOutput: slices.rotated, keys: slices.keys, values: slices.values,
      rotaryDim: headDim, rotary: "neighbours", frequencies: slices.frequencies }, shape)),
    attention.createDispatch(Object.assign({
      label: "attention", queries: slices.rotated, output: slices.attended, scoreCap: 20, window: 60 }, shape)),
    verify.createDispatch({
      label: "verify", rows, sequences, columns: spec.columns, target: slices.target, draft: slices.draft, temperature: 0.75,
      rowStarts: slices.rowStarts, tokens: slices.tokens, uniforms: slices.uniforms, draws: slices.draws,
      accepted: slices.accepted, nextTokens: slices.nextTokens }),
  ];
  const timestamps = device.createQuerySet({ type: "timestamp", count: 6 });
  const encoder = device.createCommandEncoder({ label: "draft step" });
  dispatches.forEach((d, i) => d.encode(encoder, {
    querySet: timestamps, beginningOfPassWriteIndex: 2 * i, endOfPassWriteIndex: 2 * i + 1 }, { batchSize: active }));
  device.queue.submit([encoder.finish()]);
  await device.queue.onSubmittedWorkDone();
  for (let i = 0; i < 3; ++i) assert.ok(timestamps.elapsedMs(2 * i, 2 * i + 1) > 0);
  for (const name of ["rotated", "keyCache", "valueCache", "attended", "accepted", "nextTokens"])
    fs.writeFileSync(path.join(spec.directory, `${name}.out`),
                     Buffer.from(await device.queue.readBuffer(arena.buffer, slices[name].byteOffset, slices[name].byteLength)));
  for (const d of dispatches) {
    assert.throws(() => d.encode(encoder, undefined, { batchSize: sequences + 1 }), /active sequences must be in/);
    d.destroy();
    assert.throws(() => d.encode(encoder), /was destroyed/);
  }
  console.log("host_gpu_cache ok");
}
main().catch((e) => { console.error(e); process.exit(1); });
